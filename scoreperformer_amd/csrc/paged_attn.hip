// Attention of one new row per request over its paged key / value cache (the serving form of spn_attn_fwd: causal, one query).
//   o[r, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(s_j - max s),   s_j = scale q[r, h] . k_j - slope_h (len_r - 1 - j)
// over the rows j < len_r that lie on a page; a request without any has zeros.
//
// Every cached row is read once: 2 * kvh * 64 * sizeof(T) bytes per row against 4 * h * 64 flop -- bound by HBM for every head layout, as long
// as enough loads are in flight, and below some 10 MB by the chain length -> page id -> rows -> softmax -> sum of one workgroup (4 us).
//  * A segment (request, key head, 16 query heads of it) is one workgroup's, or is cut into parts: of a 512th of the batch's tiles, but at least
//    MIN_TILES and at most max_tiles of them, and of a 128th of the segment where that is more (a lone request of 131072 rows).  The device counts
//    the batch itself, so no length is known to the host and one long cache among short ones does not set the time; a fixed grid walks the parts, so
//    a table far wider than the lengths costs the second launch and the imbalance of the lengths.  Parts leave (max, sum, unnormalised o) in the
//    workspace; a second, small launch joins them in a fixed order.
//  * Rows travel HBM -> LDS by DMA in whole 1 KiB pieces, 16 bytes a lane, consecutive lanes on consecutive bytes.  (The layouts the matrix
//    instructions want, loaded straight into registers -- a lane per row, 64 of a row's 128 bytes at a time -- hold one CU to 37 GB/s where
//    whole pieces reach 105: the first-level cache serves four lanes of one line per clock.)  Two tiles of 8 KiB per wave, private to it: no barrier.
//  * S^T = K Q^T: a lane owns ONE query head (lane & 15) and 8 (fp32: 4) rows of the tile; o^T = V^T P^T takes P^T from those very registers.
//    K is read from LDS by rows, V by transposing reads (bf16) or one row element per lane (fp32), both without bank conflicts.
//  * The query heads of one key head are the 16 columns of the tile; fewer leave columns idle, which costs nothing; more are further segments.
//  * fp32 pools: v_mfma_f32_16x16x4_f32, products and sums in fp32.  bf16 pools: products exact, sums in fp32, and a probability enters the
//    second product as TWO bf16 terms (its rounding and the remainder): off by at most 2^-16 of it instead of 2^-8, for 5 more matrix instructions
//    per tile in a kernel that waits for memory -- the output then carries one bf16 rounding, not two.  fp32 errors are 1.3 - 1.5 times those of a
//    softmax in elementary fp32 operations (2.1e-7 against 1.5e-7 of the output, 32 x 1 .. 4096).
//  * A wave instruction takes its SIMD four clocks, so what is the same for a whole tile or walk is kept off the vector unit: page ids, their
//    checks and the addresses are scalar; the bias inside a tile is the C operand of the score product; the running maximum is compared lane by
//    lane and reduced over lanes only when it moves by more than RISE; the sum of the probabilities is one more row of the value product.
// MI355X, device time: 256 requests x 8 key heads, lengths 1 .. 4096, bf16 (1.07 GB): 180 us = 6.0 TB/s; 128 x 2 key heads, 1 .. 8192 (269 MB):
// 57 us = 4.7 TB/s; 64 multi-query, 0 .. 2048 (17 MB): 10.4 us; one of 4096 rows (1 MB): 8.3 us in two launches, one of 256: 4.2 us in one.
#include "common.h"
#include "paged_index.h"
#include "paged_split.h"

using namespace spn_paged;

namespace {

constexpr int LDO = 68;             // LDS row of a head's o: 64 + 4, so that 16 heads do not meet in one bank
constexpr float LOG2E_F = 1.4426950408889634f;
constexpr float RISE = 8.f;         // log2: probabilities up to 2^8 of the reference are carried as they are

template <typename T> constexpr int TILE = 64 / (int)sizeof(T);    // rows of a tile: 32 (bf16), 16 (fp32)

static_assert(sizeof(int4) == HDR, "header of a part");

struct PagedAttnArgs {
    const void* q; long q_rs, q_hs; const void* kp; const void* vp; const int* table; long ld; const int* lens; const float* slopes;
    void* o; long o_rs, o_hs; int R, h, kvh, W, num_pages, shift; float scale;
    int group, passes;         // query heads per key head, 16-head passes over them
    int rows;                  // heads of a partial result: min(group, 16)
    int max_tiles;             // longest part aimed at, in tiles (more where a segment would have more than MAX_PARTS of them)
    int once;                  // whole segments: do not keep the rows in the caches (cut ones: decided on the device)
    int units;                 // room for this many parts
    float* part; float* ml;    // [units][rows][64], [units][rows][2]
    int4* hdr;                 // {parts of the batch; behind paged_line_kernel also: longest part aimed at, once, parts are short; otherwise 0},
                               // [units] {request, key head and pass, parts (its first part only), 0}
    int* line;                 // batches of more than SEARCH requests: [R] parts of the requests before this one
};

// reductions over the four lanes of a head (l, l ^ 16, l ^ 32, l ^ 48): the swapped halves of two copies, no LDS crossbar
__device__ __forceinline__ float quad_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float max3(float a, float b, float c) {   // without the quieting of signalling NaNs that fmaxf puts in front of every operand
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// LDS DMA of N consecutive KiB: 16 bytes per lane and piece, piece k from base + 1024 k + off[k](lane) into LDS [lds + 1024 k ..), lane-major
// (common.h spn_dma16, with a 64-bit base instead of a buffer resource: a pool passes 4 GiB; the instruction's offset counts on both sides).  The
// compiler does not count it: whoever reads waits by hand.  NT: not kept in the caches.
template <int N, bool NT>
__device__ __forceinline__ void dma(uint32_t lds, const uint32_t* off, const char* base) {
#define SPN_LEAD "s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\t"
    if constexpr (N == 1) {
        if constexpr (NT) asm volatile(SPN_LEAD "global_load_lds_dwordx4 %1, %2 nt" :: "s"(lds), "v"(off[0]), "s"(base) : "memory");
        else asm volatile(SPN_LEAD "global_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(off[0]), "s"(base) : "memory");
    } else if constexpr (N == 2) {
        if constexpr (NT)
            asm volatile(SPN_LEAD "global_load_lds_dwordx4 %1, %3 nt\n\tglobal_load_lds_dwordx4 %2, %3 offset:0x400 nt"
                         :: "s"(lds), "v"(off[0]), "v"(off[1]), "s"(base) : "memory");
        else asm volatile(SPN_LEAD "global_load_lds_dwordx4 %1, %3\n\tglobal_load_lds_dwordx4 %2, %3 offset:0x400" :: "s"(lds), "v"(off[0]), "v"(off[1]), "s"(base) : "memory");
    } else {
        static_assert(N == 4, "pieces of one base");
        if constexpr (NT)
            asm volatile(SPN_LEAD "global_load_lds_dwordx4 %1, %5 nt\n\tglobal_load_lds_dwordx4 %2, %5 offset:0x400 nt\n\tglobal_load_lds_dwordx4 %3, %5 offset:0x800 nt\n\t"
                         "global_load_lds_dwordx4 %4, %5 offset:0xc00 nt" :: "s"(lds), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base) : "memory");
        else
            asm volatile(SPN_LEAD "global_load_lds_dwordx4 %1, %5\n\tglobal_load_lds_dwordx4 %2, %5 offset:0x400\n\tglobal_load_lds_dwordx4 %3, %5 offset:0x800\n\t"
                         "global_load_lds_dwordx4 %4, %5 offset:0xc00" :: "s"(lds), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base) : "memory");
    }
#undef SPN_LEAD
}

// The page ids of a tile's groups of UNIT rows (8 where pages have 8, else 16): the same for all lanes, so they come by scalar loads -- off the
// counter of the vector loads -- and are checked by scalar instructions.
template <typename T, int UNIT> struct Pages { static constexpr int N = TILE<T> / UNIT; int id[N]; uint32_t bad; };   // bad: bit c, group c lies on no page

// One wave's walk over some tiles of one segment: the state of the softmax of 16 heads, a head per lane & 15.  Lane (i = lane & 15, g = lane >> 4).
// E: rows of a tile that a lane holds scores of.  bf16: tile rows 8 g + 0 .. 7 (row i of score product t is tile row (i >> 2) * 8 + 4 t + (i & 3),
// so that the C registers of the two are those); fp32: 4 g + 0 .. 3.
template <typename T, int WAVES>
struct Walk {
    static constexpr bool BF = sizeof(T) == 2;
    static constexpr int E = BF ? 8 : 4, ROW = HEAD * (int)sizeof(T);
    const PagedAttnArgs& a;
    const __attribute__((address_space(4))) int* trow;   // the request's table row: constant for the launch
    const char *kb, *vb;                                 // the pools at the key head
    uint32_t page_bytes;
    int n, i, g;
    char* lds; uint32_t lds0;                            // the wave's two tiles
    uint32_t off[4], ka[4], va[4];
    bf16x8 qb[2]; f32x4 qf[4];   // Q^T operand: the one of T is used
    f32x4 c0[E / 4];             // slope * (row inside the lane's E) in units of the score product
    float c1, slope2;
    float ref;                   // log2 reference of the probabilities; -inf: nothing seen yet
    f32x4 l, o[4];               // l: sum of the probabilities (bf16: in every register; fp32: the lane's own, register 0)
                                 // o[j][r]: dimension 16 j + 4 g + r (bf16), 16 g + 4 r + j (fp32)

    static __device__ __forceinline__ uint32_t spread(uint32_t q) { return (q & 1) | ((q & 2) << 1); }

    // LDS image of a tile: rows in order, a row's chunks of 16 bytes permuted so that neither the rows read together (K) nor the rows of a
    // transposing read (V) meet in a bank.  bf16, 8 chunks: chunk c of row R at place c ^ (R & 7) ^ spread(R >> 3); fp32, 16 chunks: c ^ R.  The DMA
    // writes lane-major, so the permutation is in the lanes' global offsets; inside a row's line it costs nothing.
    __device__ __forceinline__ Walk(const PagedAttnArgs& a_, int lane, char* lds_) : a(a_), i(lane & 15), g(lane >> 4), lds(lds_) {
        lds0 = __builtin_amdgcn_readfirstlane(spn_lds_addr(lds_));
        if constexpr (BF) {
            const uint32_t R = (i >> 2) * 8 + (i & 3), f = (R & 7) ^ spread(i >> 2);
            const uint32_t Rv = g * 8 + (i >> 2), fv = (Rv & 7) ^ spread(g), cv = (i & 3) >> 1;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                off[q] = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3) ^ spread(q)) * 16);
                ka[q] = R * 128 + (g ^ f ^ (q & 1 ? 4 : 0)) * 16;                         // score product t, half s: ka[t ^ s] + 512 t
                va[q] = 4096 + Rv * 128 + ((2 * q) ^ cv ^ fv) * 16 + (i & 1) * 8;         // dimensions 16 j ..: rows 0 - 3 at va[j], 4 - 7 at va[j ^ 2] + 512
            }
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                off[q] = (lane >> 4) * 256 + (((lane & 15) ^ (4 * q + (lane >> 4))) * 16);
                ka[q] = i * 256 + ((4 * q + g) ^ i) * 16;                                 // dimensions 16 q + 4 g ..
                va[q] = 4096 + (4 * g + q) * 256 + (i ^ (4 * g + q)) * 16;                // row 4 g + q, dimensions 4 i ..
            }
        }
    }

    __device__ __forceinline__ void begin(int r, int n_, int kh, int head0, int heads) {
        n = n_;
        trow = (const __attribute__((address_space(4))) int*)(a.table + r * a.ld);
        page_bytes = (uint32_t)(a.kvh * ROW) << a.shift;
        kb = (const char*)((const T*)a.kp + row_offset(0, kh, 0, a.kvh, a.shift));
        vb = (const char*)((const T*)a.vp + row_offset(0, kh, 0, a.kvh, a.shift));
        const bool on = i < heads;                  // columns behind the heads compute on zeros and are dropped
        const bool none = fabsf(a.scale) < 1e-20f;  // scores of nothing: q counts as 0 (the bias is divided by the scale)
        const bool use = on && !none;
        const T* q = (const T*)a.q + r * a.q_rs + (long)(head0 + (on ? i : 0)) * a.q_hs;   // any alignment: element loads
        if constexpr (BF) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = q[32 * s + 8 * g + 2 * e], hi = q[32 * s + 8 * g + 2 * e + 1];
                    w[e] = use ? lo | hi << 16 : 0u;
                }
                qb[s] = __builtin_bit_cast(bf16x8, w);
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) { const float x = q[16 * s + 4 * g + e]; qf[s][e] = use ? x : 0.f; }
        }
        c1 = none ? 1.f : a.scale * LOG2E_F;
        slope2 = a.slopes ? a.slopes[head0 + (on ? i : 0)] * LOG2E_F : 0.f;
        const float per = slope2 / c1;
#pragma unroll
        for (int e = 0; e < E; ++e) c0[e >> 2][e & 3] = per * (float)e;
        ref = -__builtin_inff(); l = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // rows outside the request count as its first or last one: their loads stay on its pages, their scores are dropped
    template <int UNIT> __device__ __forceinline__ Pages<T, UNIT> pages(int t) const {
        const uint32_t at = (uint32_t)max(t, 0) * TILE<T>, last = (uint32_t)(n - 1) >> a.shift;
        Pages<T, UNIT> p;
        p.bad = 0;
#pragma unroll
        for (int c = 0; c < p.N; ++c) p.id[c] = trow[min((at + UNIT * c) >> a.shift, last)];
        return p;
    }
    // an entry that is no page: page 0's rows, masked by `bad`
    template <int UNIT> __device__ __forceinline__ void check(Pages<T, UNIT>& p) const {
#pragma unroll
        for (int c = 0; c < p.N; ++c) {
            const bool ok = page_ok(p.id[c], a.num_pages);
            p.bad |= ok ? 0u : 1u << c;
            p.id[c] = ok ? p.id[c] : 0;
        }
    }
    template <int UNIT, bool NT>
    __device__ __forceinline__ void fetch(int t, const Pages<T, UNIT>& p, uint32_t stage) const {
        constexpr int PIECES = UNIT * ROW / 1024;
        const uint32_t mask = (1u << a.shift) - 1u;
#pragma unroll
        for (int c = 0; c < p.N; ++c) {
            // (uniform by construction; said once more, because the compiler does not always see it through the loop)
            const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(p.id[c]) * page_bytes +
                                (uint32_t)__builtin_amdgcn_readfirstlane((((uint32_t)t * TILE<T> + UNIT * c) & mask) * ROW);
            dma<PIECES, NT>(lds0 + stage + c * PIECES * 1024, off + c * PIECES, kb + at);
            dma<PIECES, NT>(lds0 + stage + 4096 + c * PIECES * 1024, off + c * PIECES, vb + at);
        }
    }

    // Tiles t, t - WAVES, ... down to t0, the newest rows first.  Two tiles are on their way while one is computed; a tile's LDS is refilled as soon
    // as it has been read into registers.
    template <int UNIT, bool NT>
    __device__ __forceinline__ void run(int t, int t0) {
        if (t < t0) return;
        Pages<T, UNIT> now = pages<UNIT>(t), next = pages<UNIT>(t - WAVES), then = pages<UNIT>(t - 2 * WAVES);
        check(now);
        fetch<UNIT, NT>(t, now, 0);
        check(next);
        if (t - WAVES >= t0) fetch<UNIT, NT>(t - WAVES, next, STAGE);
        uint32_t stage = 0;
        for (;;) {
            const bool more = t - WAVES >= t0;
            // the 8 youngest loads are the next tile's (loads return in order; others in between only make the wait longer)
            if (more) asm volatile("s_waitcnt vmcnt(8)" ::: "memory"); else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const char* st = lds + stage;
            f32x4 s[E / 4];
            bf16x8 vb8[4]; f32x4 vf[4];
            if constexpr (BF) {
                s[0] = c0[0]; s[1] = c0[1];
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(st + ka[tt ^ e] + tt * 512), qb[e], s[tt], 0, 0, 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
                    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(st + va[j]));
                    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(st + va[j ^ 2] + 512));
                    vb8[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                }
            } else {
                s[0] = c0[0];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f32x4 k = *reinterpret_cast<const f32x4*>(st + ka[e]);
#pragma unroll
                    for (int f = 0; f < 4; ++f) s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[f], qf[e][f], s[0], 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) vf[e] = *reinterpret_cast<const f32x4*>(st + va[e]);
            }
            check(then);
            if (t - 2 * WAVES >= t0) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this tile has been read
                fetch<UNIT, NT>(t - 2 * WAVES, then, stage);
            }
            const Pages<T, UNIT> later = pages<UNIT>(t - 3 * WAVES);   // behind the LDS reads: scalar loads share their counter
            if constexpr (BF) weigh(vb8, s, t, now); else weigh(vf, s, t, now);
            if (!more) return;
            t -= WAVES; stage ^= STAGE;
            now = next; next = then; then = later;
        }
    }

    // softmax weights of the lane's E rows and their share of o
    template <typename V, int UNIT>
    __device__ __forceinline__ void weigh(V (&v)[4], const f32x4 (&s)[E / 4], int t, const Pages<T, UNIT>& pg) {
        const int row0 = t * TILE<T> + g * E;
        const bool unset = ref == -__builtin_inff();
        const float base = __builtin_fmaf(slope2, (float)(row0 - (n - 1)), unset ? 0.f : -ref);
        float p[E];
#pragma unroll
        for (int e = 0; e < E; ++e) p[e] = __builtin_fmaf(c1, s[e >> 2][e & 3], base);
        if (part_filled(t, TILE<T>, n) || pg.bad) {   // rows behind the length or on no page: no weight, and no bit of theirs in the product
            const bool ok = !(pg.bad >> (g * E / UNIT) & 1);
#pragma unroll
            for (int e = 0; e < E; ++e) p[e] = ok && row0 + e < n ? p[e] : -__builtin_inff();
            if constexpr (BF) {
                u32x4 keep;
#pragma unroll
                for (int e = 0; e < 4; ++e) keep[e] = !ok || row0 + 2 * e >= n ? 0u : row0 + 2 * e + 1 >= n ? 0xffffu : 0xffffffffu;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = __builtin_bit_cast(V, __builtin_bit_cast(u32x4, v[j]) & keep);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int f = 0; f < 4; ++f) v[e][f] = ok && row0 + e < n ? v[e][f] : 0.f;
            }
        }
        float own = max3(p[0], p[1], max3(p[2], p[3], p[3]));
        if constexpr (BF) own = max3(own, p[4], max3(p[5], p[6], p[7]));
        if (__any(own > (unset ? -__builtin_inff() : RISE))) {   // rare: the walk goes from the newest rows, where the bias is largest, to the oldest
            const float up = quad_max(own);
            if (up > (unset ? -__builtin_inff() : RISE)) {
                const float c = unset ? 0.f : __builtin_amdgcn_exp2f(-up);   // (unset: nothing but zeros to scale)
                ref = unset ? up : ref + up;
#pragma unroll
                for (int e = 0; e < E; ++e) p[e] -= up;
                l *= c;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] *= c;
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) p[e] = __builtin_amdgcn_exp2f(p[e]);
        if constexpr (BF) {
            u32x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t w = pack_bf2(p[2 * e], p[2 * e + 1]);
                asm("" : "+v"(w));   // (the low half by a shift of the pair, not by a second conversion)
                hi[e] = w;
                lo[e] = pack_bf2(p[2 * e] - __uint_as_float(w << 16), p[2 * e + 1] - __uint_as_float(w & 0xffff0000u));
            }
            const bf16x8 ph = __builtin_bit_cast(bf16x8, hi), pl = __builtin_bit_cast(bf16x8, lo);
            const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
            l = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, ph, l, 0, 0, 0);
            l = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pl, l, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[j], ph, o[j], 0, 0, 0);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[j], pl, o[j], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                l[0] += p[e];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e][j], p[e], o[j], 0, 0, 0);
            }
        }
    }

    // (reference, sum, o) of the 16 heads over the wave's own tiles, when it has used them up: [16][LDO] floats, 16 references, 16 sums
    __device__ __forceinline__ void leave() {
        float* so = reinterpret_cast<float*>(lds) + i * LDO;
        const float sum = BF ? l[0] : quad_sum(l[0]);
        if (g == 0) { reinterpret_cast<float*>(lds)[HEADS * LDO + i] = ref; reinterpret_cast<float*>(lds)[HEADS * LDO + HEADS + i] = sum; }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (BF) *reinterpret_cast<f32x4*>(so + 16 * q + 4 * g) = o[q];
            else *reinterpret_cast<f32x4*>(so + 16 * g + 4 * q) = f32x4{o[0][q], o[1][q], o[2][q], o[3][q]};
        }
    }
};

template <typename T>
__device__ __forceinline__ void store4(T* to, const float (&v)[4]) {   // any alignment
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 2) to[e] = f2bf(v[e]); else to[e] = v[e];
    }
}
// weight of a partial result with reference m under the common one
__device__ __forceinline__ float under(float m, float M) { return m == -__builtin_inff() ? 0.f : m == M ? 1.f : __builtin_amdgcn_exp2f(m - M); }

// Inclusive sum over the wave's lanes (row shifts by 1, 2, 4, 8, then the rows' last lanes into the rows behind).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}

template <typename T> __device__ __forceinline__ int tiles_in(int rows) { return tiles_of(rows, TILE<T>); }
__device__ __forceinline__ int rows_at(const PagedAttnArgs& a, int r) { return rows_of(a.lens[r], a.W, a.shift); }

// tiles [t0, t1) of segment hp (key head and 16-head pass) of request r, which holds n rows; parts: into how many the segment is cut
struct Part { int r, n, hp, t0, t1, part, parts; };

// One part of one segment by WAVES waves (threads tid, LDS smem): their walks, and their results put together -- into the output, or (slot >= 0) into
// a partial result.
template <typename T, int WAVES>
__device__ __forceinline__ void do_part(const PagedAttnArgs& a, char (*smem)[2 * STAGE], int tid, const Part& p, bool once, long slot) {
    const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r = p.r;
    const int kh = p.hp / a.passes, first = (p.hp - kh * a.passes) * HEADS, heads = min(HEADS, a.group - first), head0 = kh * a.group + first;
    Walk<T, WAVES> wk(a, lane, smem[w]);
    wk.begin(r, p.n, kh, head0, heads);
    if (a.shift == 3) { if (once) wk.template run<8, true>(p.t1 - 1 - w, p.t0); else wk.template run<8, false>(p.t1 - 1 - w, p.t0); }
    else { if (once) wk.template run<16, true>(p.t1 - 1 - w, p.t0); else wk.template run<16, false>(p.t1 - 1 - w, p.t0); }
    wk.leave();
    if constexpr (WAVES == 1) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); else __syncthreads();
    const int d = (tid & 15) * 4;   // 16 threads a head, 4 dimensions each
    for (int hd = tid >> 4; hd < heads; hd += 4 * WAVES) {
        float M = -__builtin_inff(), L = 0.f, O[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < WAVES; ++u) M = fmaxf(M, reinterpret_cast<const float*>(smem[u])[HEADS * LDO + hd]);
#pragma unroll
        for (int u = 0; u < WAVES; ++u) {
            const float* su = reinterpret_cast<const float*>(smem[u]);
            const float c = under(su[HEADS * LDO + hd], M);
            const f32x4 ov = *reinterpret_cast<const f32x4*>(su + hd * LDO + d);
            L += c * su[HEADS * LDO + HEADS + hd];
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] += c * ov[e];
        }
        if (slot < 0) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] = L == 0.f ? 0.f : O[e] * inv;
            store4((T*)a.o + r * a.o_rs + (long)(head0 + hd) * a.o_hs + d, O);
        } else {
            const long at = slot * a.rows + hd;
            *reinterpret_cast<f32x4*>(a.part + at * HEAD + d) = f32x4{O[0], O[1], O[2], O[3]};
            if (d == 0) { a.ml[2 * at] = M; a.ml[2 * at + 1] = L; }
        }
    }
}

// Four parts by four waves: a wave each where all are short, otherwise one after the other by all four.  A short part costs its latency, not its
// bytes: 8000 segments of up to 100 rows 112 -> 55 us.
constexpr int SHORT = 24;   // tiles
template <typename T, typename At, typename Done>
__device__ __forceinline__ void do_four(const PagedAttnArgs& a, char (*smem)[2 * STAGE], int* tiles, int tid, int u, int all, bool once, const At& at,
                                        const Done& done) {
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), own = min(u + w, all - 1);
    const Part mine = at(own);
    if ((tid & 63) == 0) tiles[w] = mine.t1 - mine.t0;
    __syncthreads();
    const int longest = max(max(tiles[0], tiles[1]), max(tiles[2], tiles[3]));
    if (__builtin_amdgcn_readfirstlane(longest) <= SHORT) {
        if (u + w < all) {
            do_part<T, 1>(a, smem + w, tid & 63, mine, once, mine.parts > 1 ? own : -1);
            if ((tid & 63) == 0) done(own, mine);
        }
    } else {
        for (int k = 0; k < 4 && u + k < all; ++k) {
            if (k) __syncthreads();
            const Part p = at(u + k);
            do_part<T, 4>(a, smem, tid, p, once, p.parts > 1 ? u + k : -1);
            if (tid == 0) done(u + k, p);
        }
    }
}

// A workgroup takes a whole segment.
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_attn_whole_kernel(PagedAttnArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[WAVES][2 * STAGE];
    const int H = a.kvh * a.passes, r = blockIdx.x / H, n = rows_at(a, r);
    do_part<T, WAVES>(a, smem, threadIdx.x, Part{r, n, (int)blockIdx.x - r * H, 0, tiles_in<T>(n), 0, 1}, a.once, -1);
}

// Many requests: the line of parts by one workgroup in front, instead of by every wave (in wide tables, by every wave / in front: 16384 requests
// of up to 100 rows 343 / 95 us, 4096 82 / 29, 500 15.0 / 11.5, 256 of up to 1000 19.1 / 20.8: hence SEARCH).
constexpr int LINE_T = 1024;
template <typename T>
__global__ __launch_bounds__(LINE_T) void paged_line_kernel(PagedAttnArgs a) {
    __shared__ long s_sum[LINE_T / 64];
    __shared__ int s_end[2][LINE_T / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, H = a.kvh * a.passes;
    long mine = 0;
#pragma unroll 4
    for (int r = tid; r < a.R; r += LINE_T) mine += tiles_in<T>(rows_at(a, r));
#pragma unroll
    for (int d = 32; d; d >>= 1) mine += __shfl_xor(mine, d, 64);
    if (lane == 0) s_sum[w] = mine;
    __syncthreads();
    long total = 0;
    for (int i = 0; i < LINE_T / 64; ++i) total += s_sum[i];
    total *= H;
    const int most = most_of(total, a.max_tiles);
    int carry = 0;   // (the same in all threads)
    for (int r0 = 0, k = 0; r0 < a.R; r0 += LINE_T, k ^= 1) {
        const int r = r0 + tid, here = r < a.R ? H * parts_of(tiles_in<T>(rows_at(a, r)), most) : 0, to = wave_scan(here);
        if (lane == 63) s_end[k][w] = to;
        __syncthreads();   // (one a round: the other half of s_end is still being read)
        int before = 0, round = 0;
        for (int i = 0; i < LINE_T / 64; ++i) { const int e = s_end[k][i]; before += i < w ? e : 0; round += e; }
        if (r < a.R) a.line[r] = carry + before + to - here;
        carry += round;
    }
    if (tid == 0) a.hdr[0] = int4{min(carry, a.units), most, total * STAGE >= ONCE, total <= (long)carry * (SHORT / 2)};
}

// Segments cut into parts (paged_split.h most_of, parts_of): the parts of all segments stand in one line, of which workgroup g takes
// number g, g + G, ...  (four at a time where there are enough of them, and short).  SEARCHED: the line was drawn by the kernel above; otherwise
// every wave draws it for itself (a lane: every 64th stretch of requests; no barrier, no LDS, no launch).
template <typename T, bool SEARCHED>
__global__ __launch_bounds__(256, 2) void paged_attn_cut_kernel(PagedAttnArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[4][2 * STAGE];
    __shared__ int s_tiles[4];
    const int tid = threadIdx.x, lane = tid & 63, H = a.kvh * a.passes;
    const int per = (a.R + 63) / 64;
    int all, most, first = 0, incl = 0, units = 0;
    bool once, is_short;
    if constexpr (SEARCHED) {
        const int4 head = a.hdr[0];
        all = __builtin_amdgcn_readfirstlane(head.x); most = __builtin_amdgcn_readfirstlane(head.y);
        once = __builtin_amdgcn_readfirstlane(head.z); is_short = __builtin_amdgcn_readfirstlane(head.w);
    } else {
        const int q0 = min(a.R, lane * per), q1 = min(a.R, q0 + per);   // this lane's requests
        first = q0 < q1 ? rows_at(a, q0) : 0;
        long mine = tiles_in<T>(first);
        for (int q = q0 + 1; q < q1; ++q) mine += tiles_in<T>(rows_at(a, q));
        // in two halves of 32 bits: table capacities pass 2^32 tiles before memory does
        const long total = H * (((long)__builtin_amdgcn_readlane(wave_scan((int)(mine >> 16)), 63) << 16) +
                                (uint32_t)__builtin_amdgcn_readlane(wave_scan((int)(mine & 0xffff)), 63));
        most = most_of(total, a.max_tiles);
        once = total * STAGE >= ONCE;
        units = q0 < q1 ? H * parts_of(tiles_in<T>(first), most) : 0;
        for (int q = q0 + 1; q < q1; ++q) units += H * parts_of(tiles_in<T>(rows_at(a, q)), most);
        incl = wave_scan(units);
        all = min(__builtin_amdgcn_readlane(incl, 63), a.units);
        is_short = total <= (long)all * (SHORT / 2);
        if (blockIdx.x == 0 && tid == 0) a.hdr[0] = int4{all, 0, 0, 0};
    }
    const auto at = [&](int u) {
        Part p;
        int off = u;
        if constexpr (SEARCHED) {   // the last request that begins at or before u: 64 candidates at a time
            int base = 0, span = a.R;
            while (span > 1) {
                const int step = (span + 63) >> 6;
                const bool in = lane * step < span;
                const int from = a.line[base + (in ? lane * step : 0)], k = 63 - __builtin_clzll(__ballot(in && from <= u) | 1);
                base += k * step; span = min(step, span - k * step);
            }
            p.r = base; p.n = __builtin_amdgcn_readfirstlane(rows_at(a, base)); off -= __builtin_amdgcn_readfirstlane(a.line[base]);
        } else {
            const int from = __builtin_ctzll(__ballot(incl > u));
            off -= __builtin_amdgcn_readlane(incl - units, from);
            p.r = from * per; p.n = __builtin_amdgcn_readlane(first, from);
            // more than 64 requests: those of the lane that was found, a lane each (SEARCH / 64 at most)
            if (per > 1) {
                const int q = p.r + lane, rows = lane < per && q < a.R ? rows_at(a, q) : 0;
                const int here = lane < per && q < a.R ? H * parts_of(tiles_in<T>(rows), most) : 0, to = wave_scan(here);
                const unsigned long long found = __ballot(to > off);
                const int k = found ? __builtin_ctzll(found) : 0;
                p.r += k; p.n = __builtin_amdgcn_readlane(rows, k);
                off -= __builtin_amdgcn_readlane(to - here, k);
            }
        }
        p.parts = parts_of(tiles_in<T>(p.n), most);
        // (the bounds hold by themselves unless the lengths change while this runs; then the result is lost, but no access goes astray)
        p.hp = max(0, min(off / p.parts, H - 1)); p.part = max(0, min(off - p.hp * p.parts, p.parts - 1));
        const int tiles = tiles_in<T>(p.n);
        p.t0 = (int)((long)tiles * p.part / p.parts); p.t1 = (int)((long)tiles * (p.part + 1) / p.parts);
        return p;
    };
    const auto done = [&](int u, const Part& p) { a.hdr[1 + u] = int4{p.r, p.hp, p.part == 0 && p.parts > 1 ? p.parts : 0, 0}; };
    if (all >= 4 * RESIDENT && is_short) {
        for (int u = 4 * blockIdx.x; u < all; u += 4 * gridDim.x) {
            do_four<T>(a, smem, s_tiles, tid, u, all, once, at, done);
            __syncthreads();   // the tiles of the next parts go where these results were
        }
    } else {
        for (int u = blockIdx.x; u < all; u += gridDim.x) {
            const Part p = at(u);
            do_part<T, 4>(a, smem, tid, p, once, p.parts > 1 ? u : -1);
            if (tid == 0) done(u, p);
            __syncthreads();
        }
    }
}

// Joins the parts of a segment that was cut: slots g .. g + parts - 1, in a fixed order.  JOIN_HEADS heads a block; 16 lanes (4 dimensions each) take
// every 8th part of a head, eight of them in flight.  3.5 us for a few parts (a launch is 2.5), about 6 us for 128 parts of 8 heads.
constexpr int JOIN_HEADS = 2, JOIN_SUBS = 16 / JOIN_HEADS;
template <typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
    __shared__ float s_o[16][LDO], s_m[16], s_l[16];
    int4 cut = a.hdr[1 + blockIdx.x];   // (written or not: asked for together with the count)
    const int all = min(a.hdr[0].x, a.units), grp = threadIdx.x >> 4, d = (threadIdx.x & 15) * 4, sub = grp % JOIN_SUBS;
    const int hd = blockIdx.y * JOIN_HEADS + grp / JOIN_SUBS;
    for (int g = blockIdx.x; g < all; g += gridDim.x) {
        if (g != (int)blockIdx.x) cut = a.hdr[1 + g];
        if (cut.z == 0) continue;
        const int parts = min(cut.z, all - g);
        const int kh = cut.y / a.passes, first = (cut.y - kh * a.passes) * HEADS, heads = min(HEADS, a.group - first), head0 = kh * a.group + first;
        float M = -__builtin_inff(), L = 0.f;
        f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
        if (hd < heads) {
            const float* ml = a.ml + 2 * ((long)g * a.rows + hd);
            const float* po = a.part + ((long)g * a.rows + hd) * HEAD + d;
            constexpr int U = 8;
            for (int p = sub; p < parts; p += JOIN_SUBS * U) {
                float m[U], l[U];
                f32x4 o[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const long at = (long)min(p + u * JOIN_SUBS, parts - 1) * a.rows;
                    m[u] = ml[2 * at]; l[u] = ml[2 * at + 1];
                    o[u] = *reinterpret_cast<const f32x4*>(po + at * HEAD);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (p + u * JOIN_SUBS >= parts) { m[u] = -__builtin_inff(); l[u] = 0.f; o[u] = f32x4{0.f, 0.f, 0.f, 0.f}; }
                    const float mn = fmaxf(M, m[u]), c = M == mn ? 1.f : __builtin_amdgcn_exp2f(M - mn), b = under(m[u], mn);
                    L = L * c + l[u] * b; M = mn;
#pragma unroll
                    for (int e = 0; e < 4; ++e) O[e] = O[e] * c + o[u][e] * b;
                }
            }
        }
        __syncthreads();   // (the previous one has been read)
        *reinterpret_cast<f32x4*>(&s_o[grp][d]) = O;
        if (d == 0) { s_m[grp] = M; s_l[grp] = L; }
        __syncthreads();
        if (sub == 0 && hd < heads) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            M = -__builtin_inff(); L = 0.f;
#pragma unroll
            for (int u = 0; u < JOIN_SUBS; ++u) M = fmaxf(M, s_m[grp + u]);
#pragma unroll
            for (int u = 0; u < JOIN_SUBS; ++u) {
                const float c = under(s_m[grp + u], M);
                L += c * s_l[grp + u];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += c * s_o[grp + u][d + e];
            }
            const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = L == 0.f ? 0.f : v[e] * inv;
            store4((T*)a.o + cut.x * a.o_rs + (long)(head0 + hd) * a.o_hs + d, v);
        }
    }
}

int page_shift(int page) {
    for (int s = 3; s <= 12; ++s) if (page == 1 << s) return s;
    return -1;
}

template <typename T, int WAVES>
void launch_whole(const PagedAttnArgs& a, long segments, hipStream_t stream) {
    hipLaunchKernelGGL((paged_attn_whole_kernel<T, WAVES>), dim3((unsigned)segments), dim3(64 * WAVES), 0, stream, a);
}
template <typename T>
int launch(const PagedAttnArgs& a, const Split& s, hipStream_t stream) {
    if (s.waves == 8) launch_whole<T, 8>(a, s.units, stream);
    else if (s.waves == 4) launch_whole<T, 4>(a, s.units, stream);
    else if (s.waves == 2) launch_whole<T, 2>(a, s.units, stream);
    else {
        const unsigned grid = s.units < GRID ? (unsigned)s.units : GRID;
        if (a.R > SEARCH) {
            hipLaunchKernelGGL(paged_line_kernel<T>, dim3(1), dim3(LINE_T), 0, stream, a);
            SPN_LAUNCH_CHECK();
            hipLaunchKernelGGL((paged_attn_cut_kernel<T, true>), dim3(grid), dim3(256), 0, stream, a);
        } else hipLaunchKernelGGL((paged_attn_cut_kernel<T, false>), dim3(grid), dim3(256), 0, stream, a);
        SPN_LAUNCH_CHECK();
        hipLaunchKernelGGL(paged_join_kernel<T>, dim3(grid, cdiv(a.rows, JOIN_HEADS)), dim3(256), 0, stream, a);
    }
    SPN_LAUNCH_CHECK();
    return SPN_OK;
}

}  // namespace

extern "C" size_t spn_paged_attn_workspace_bytes(int R, int h, int kvh, int W, int page, int dtype) {
    const int shift = page_shift(page);
    if (shift < 0 || !sizes_ok(R, h, kvh, W, shift)) return 0;   // refused by the call itself
    return scratch_of(split_of(R, h, kvh, W, shift, dtype == 1 ? 2 : 4), R);
}

extern "C" int spn_paged_attn(const void* q, long q_rs, long q_hs, const void* k_pages, const void* v_pages, int dtype, const int* block_table, long bt_ld,
                              const int* lens, const float* slopes, void* o, long o_rs, long o_hs, int R, int h, int kvh, int W, int num_pages,
                              int page, float scale, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const int shift = page_shift(page);
    SPN_REQUIRE(q && k_pages && v_pages && block_table && lens && o, "spn_paged_attn: null buffer");
    SPN_REQUIRE(dtype == 0 || dtype == 1, "spn_paged_attn: dtype codes are 0 (fp32) and 1 (bf16)");
    SPN_REQUIRE(shift >= 0, "spn_paged_attn: the page size must be a power of two in [8, 4096]");
    SPN_REQUIRE(num_pages > 0 && bt_ld >= W && sizes_ok(R, h, kvh, W, shift), "spn_paged_attn: bad sizes");
    SPN_REQUIRE(((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) == 0, "spn_paged_attn: pages must be 16-byte aligned");
    const Split s = split_of(R, h, kvh, W, shift, dtype == 1 ? 2 : 4);
    const size_t need = scratch_of(s, R);
    SPN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                "spn_paged_attn: the workspace is too small or not 16-byte aligned (spn_paged_attn_workspace_bytes)");
    PagedAttnArgs a{q, q_rs, q_hs, k_pages, v_pages, block_table, bt_ld, lens, slopes, o, o_rs, o_hs, R, h, kvh, W, num_pages, shift, scale,
                    h / kvh, s.passes, s.rows, s.max_tiles, s.once, (int)s.units, nullptr, nullptr, nullptr, nullptr};
    if (need) { a.hdr = (int4*)workspace; a.part = (float*)(a.hdr + 1 + s.units); a.ml = a.part + s.units * s.rows * HEAD; a.line = (int*)(a.ml + s.units * s.rows * 2); }
    return dtype == 1 ? launch<bf16_t>(a, s, stream) : launch<float>(a, s, stream);
}
