// How the attention over the paged cache (paged_attn.hip) divides a batch: plain integer functions, shared by the kernels and by the host-compiled
// check of their bounds (tests/test_paged_cpu.py builds this header with the host compiler).
#pragma once
#include <stddef.h>
#include "paged_index.h"

namespace spn_paged {

constexpr int HEADS = 16;           // query heads of a segment
constexpr int STAGE = 8192;         // bytes of a tile: 4 KiB of keys, 4 KiB of values
constexpr int MIN_TILES = 4;        // least tiles of a part (a tile per wave; 2: the same, 8: 1 x 4096 rows 8.9 -> 8.2 us the other way)
constexpr int TARGET = 512;         // parts the batch is cut into, beside one per segment (1024: the same within 2 %)
constexpr int MAX_TILES = 64;       // longest part aimed at where the batch is larger (32: 256 x 4096 rows 182 -> 196 us, 128: 186)
constexpr int RESIDENT = 512;       // workgroups of 4 waves that run at once: two on a compute unit, by their LDS
constexpr unsigned GRID = 2 * RESIDENT;   // workgroups of a cut batch
constexpr int MAX_PARTS = 128;      // parts of a segment (one of 131072 rows, 256: 18.9 us, 128: 17.2, 64: 20.8 when a tile cost a tenth more)
constexpr int SEARCH = 256;         // requests from which the line of parts is drawn by a workgroup in front (times at paged_line_kernel)
constexpr size_t HDR = 16;          // bytes of a part's header

constexpr long ONCE = 64L << 20;   // bytes of rows from which they are not kept in the caches (Infinity Cache: 256 MiB; a step walks every layer's cache
                                   // before it is back at this one).  1.07 GB: 195 -> 177 us; 17 MB, three pools in turn: 11.4 -> 13.3 us, hence the bound

// tiles of `tile` rows that 0 .. 2^31 - 1 rows take, and whether tile t of them is not filled to its end: no sum passes the type
SPN_HD int tiles_of(int rows, int tile) { return (int)(((uint32_t)rows + (uint32_t)tile - 1u) / (uint32_t)tile); }
SPN_HD bool part_filled(int t, int tile, int rows) { return rows - t * tile < tile; }

// parts of a segment of `tiles` tiles, none above `most` tiles unless there would be more than MAX_PARTS
SPN_HD int parts_of(int tiles, int most) {
    const int parts = (int)(((uint32_t)tiles + (uint32_t)most - 1u) / (uint32_t)most);
    return parts < 1 ? 1 : parts < MAX_PARTS ? parts : MAX_PARTS;
}

// the longest part aimed at in a batch of `total` tiles
SPN_HD int most_of(long total, int max_tiles) {
    const long even = (total + TARGET - 1) / TARGET, most = even < MIN_TILES ? MIN_TILES : even;
    return (int)(most < max_tiles ? most : max_tiles);
}

// the sizes a call may have: rows of a request, table entries and bytes of a page stay in 32 bits, segments in the grid
inline bool sizes_ok(int R, int h, int kvh, int W, int shift) {
    return R > 0 && h > 0 && kvh > 0 && h % kvh == 0 && W > 0 && ((long)W << shift) < (1L << 31) && (long)R * W < (1L << 31) && (long)R * h < (1L << 21) &&
           ((long)kvh * HEAD * 4 << shift) < (1L << 32);
}

struct Split { long units; int waves; int passes, rows, max_tiles, once; };   // waves: of a workgroup that takes a whole segment; 0: cut
inline Split split_of(int R, int h, int kvh, int W, int shift, int esize) {
    Split s;
    const int group = h / kvh;
    s.passes = (group + HEADS - 1) / HEADS; s.rows = group < HEADS ? group : HEADS;
    const long segments = (long)R * kvh * s.passes, cap = (long)W << shift, bytes = cap * HEAD * 2 * esize, tiles = (bytes + STAGE - 1) / STAGE;
    // Whole segments, one launch instead of two: a lone workgroup of 8 waves reads 105 GB/s (fp32, bound by its matrix instructions: 56), the machine
    // about 5 TB/s, the second launch costs some 6 us of device and host time, so with tables filled by half
    //   bytes / rate  <=  segments * bytes / 2 / 5 TB/s + 6 us,
    // and never where one full table among short ones would take long by itself (1 MiB: 10 us for 4096 rows of a bf16 key head, 19 for 2048 of fp32).
    // Measured, whole / cut: 64 x 2048 rows 10.3 / 13.5 us, 1 x 4096 13.6 / 8.2, 16 x 512 5.1 / 8.2, 39 segments of 1001 fp32 rows 14.5 / 10.7,
    // 2048 segments of up to 4096 rows 176 / 184.
    const long rate = esize == 2 ? 105 : 56;   // bytes per ns
    const bool whole = bytes <= (1L << 20) && bytes * (10000 - rate * segments) <= 6000 * rate * 10000;
    // waves: 8 where the segments do not fill the machine.  Where they do, their lengths decide, which the host does not know: 8 waves serve long rows
    // best (2048 segments of up to 4096 rows, 2 / 4 / 8 waves: 193, 180, 176 us), 2 waves short ones (8000 of up to 100: 30, 50, 89; 2048 of up to
    // 500: 26, 28, 38; of up to 1000: 45, 43, 51), so the width of the tables is the hint and 8 is left out
    s.waves = !whole ? 0 : segments >= 4 * RESIDENT ? (tiles > 64 ? 4 : 2) : segments > 256 ? 4 : tiles > 8 ? 8 : 4;
    s.once = segments * bytes >= 2 * ONCE;   // tables filled by half
    // the longest part: MAX_TILES, or what keeps the workspace -- all tables full -- to 8192 parts
    const long full = segments * tiles, most = (full + 8191) / 8192;
    const long part = most < MAX_TILES ? MAX_TILES : most, whole_one = tiles < MAX_TILES ? MAX_TILES : tiles;
    s.max_tiles = (int)(part < whole_one ? part : whole_one);   // (never more than a full segment: `part` passes 2^31 where tables of 2^30 rows have 2^20 segments)
    // parts on the device: at most tiles / most + 1 for each segment, with most >= MIN_TILES and most >= min(max_tiles, all tiles / TARGET)
    long units = full / part;
    units = (units < TARGET ? TARGET : units) + segments;
    const long finest = segments * ((tiles + MIN_TILES - 1) / MIN_TILES);
    s.units = whole ? segments : units < finest ? units : finest;
    return s;
}

inline size_t scratch_of(const Split& s, int R) {
    if (s.waves) return 0;
    return (size_t)s.units * ((size_t)s.rows * (HEAD + 2) * sizeof(float) + HDR) + HDR + (R > SEARCH ? R * sizeof(int) : 0);
}

}  // namespace spn_paged
