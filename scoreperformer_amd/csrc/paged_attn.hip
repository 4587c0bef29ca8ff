// Attention of one new row per request over its paged key / value cache (the serving form of spn_attn_fwd: causal, one query).
//   o[r, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(s_j - max s),   s_j = scale q[r, h] . k_j - slope_h (len_r - 1 - j)
// over the rows j < len_r that lie on a page; a request without any has zeros.
//
// Every cached row is read once: 2 * kvh * 64 * sizeof(T) bytes per row against 4 * h * 64 flop -- bound by HBM for every head layout, as long
// as enough loads are in flight.  What follows from that:
//  * Work is cut by ROWS, not by requests: the batch's tiles of 32 rows (request-major, then key head) form one line, and workgroup g of G takes
//    the g-th G-th of it, wherever requests begin and end.  One long cache among short ones, or a table far wider than the lengths, costs
//    nothing; no length is known to the host.  A request that lies in one workgroup is finished there; one that is cut leaves partial sums (max,
//    sum, unnormalised o) in the workspace and a second, small launch joins them in a fixed order.
//  * One wave = one tile at a time, straight from HBM to registers: the matrix products are arranged so that neither operand needs a transpose
//    through LDS.  S^T = K Q^T (rows of K are the A operand as they lie in memory; a lane owns ONE head, lane & 15, and 8 rows of the tile),
//    o^T = V^T P^T (P^T is already the B operand in that layout; V rows arrive as 4 dimensions x 8 rows per lane and 16 byte permutes turn the
//    8 rows of a dimension into one register quad).  The next tile's loads are issued before the current tile is computed, its page ids one
//    tile earlier still.
//  * The query heads of one key head are the 16 columns of the tile; fewer than 16 leave columns idle, which costs nothing (bound by bytes);
//    more are further passes.
//  * fp32 pools: the same layouts through v_mfma_f32_16x16x4_f32, products and sums in fp32.  bf16 pools: products exact, sums in fp32, and a
//    probability enters the second product as TWO bf16 terms (its rounding and the remainder): 2^-17 instead of 2^-9 of it, for 4 more matrix
//    instructions per tile in a kernel that waits for memory -- the output then carries one bf16 rounding, not two.
#include "common.h"
#include "paged_index.h"

using namespace spn_paged;

namespace {

constexpr int TILE = 32;       // rows per tile
#ifndef PA_MIN_TILES
#define PA_MIN_TILES 4
#endif
#ifndef PA_TARGET
#define PA_TARGET 512
#endif
#ifndef PA_WAVES
#define PA_WAVES 4
#endif
#ifndef PA_MAX_TILES
#define PA_MAX_TILES 32
#endif
constexpr int WAVES = PA_WAVES, MIN_TILES = PA_MIN_TILES, TARGET = PA_TARGET, MAX_TILES = PA_MAX_TILES;

constexpr int HEADS = 16;      // query heads per pass
constexpr int LDO = 68;        // LDS row of a head's o: 64 + 4, so that 16 heads do not meet in one bank
constexpr float LOG2E_F = 1.4426950408889634f;

struct PagedAttnArgs {
    const void* q; long q_rs, q_hs; const void* kp; const void* vp; const int* table; long ld; const int* lens; const float* slopes;
    void* o; long o_rs, o_hs; int R, h, kvh, W, num_pages, shift; float scale;
    int group, passes;         // query heads per key head, 16-head passes over them
    int rows;                  // heads of a partial result: min(group, 16)
    int max_tiles;             // most tiles of a part
    int once;                  // rows are not kept in the caches: see launch
    float* part; float* ml; int4* hdr;   // [G][rows][64], [G][rows][2], [G] {request, key head and pass, parts (its first part only), 0}
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

// A tile's rows as they arrive.  Lane (i = lane & 15, g = lane >> 4).  K: tile row (i >> 2) * 8 + 4 t + (i & 3) for t = 0, 1, so that the C
// registers of the two products hold rows g * 8 .. g * 8 + 7.  V: rows g * 8 + 0 .. 7, dimensions 4 i .. 4 i + 3.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <typename T> struct Tile;
template <> struct Tile<bf16_t> { typedef u32x4 K; typedef u32x2 V; static constexpr int PER = 2; K k[2][2]; V v[8]; };   // k[t][s]: dimensions 32 s + 8 g ..
template <> struct Tile<float> { typedef f32x4 K; typedef f32x4 V; static constexpr int PER = 4; K k[2][4]; V v[8]; };    // k[t][s]: dimensions 16 s + 4 g ..

// The page ids of a tile's four groups of 8 rows (a page holds at least 8): the same for all lanes, so they come by scalar loads -- off the
// counter of the vector loads, whose order they would otherwise take part in -- and are checked by scalar instructions.
struct Pages { int id[4]; bool ok[4]; };

// One wave's walk over some tiles of one (request, key head): the state of the softmax of 16 heads, a head per lane & 15.  The loop is bound by
// instruction issue where few workgroups run (a wave instruction takes a SIMD four clocks), so what is the same for a whole tile or a whole walk
// is kept out of the vector unit: page ids and checks are scalar, the bias inside a tile is the C operand of the score product, the running
// maximum is compared lane by lane and reduced over lanes only when it moves by more than RISE, the sum of the probabilities is one more row of the
// value product.
constexpr float RISE = 8.f;   // log2: probabilities up to 2^8 of the reference are carried as they are

template <typename T>
struct Walk {
    typedef Tile<T> X;
    const PagedAttnArgs& a;
    const __attribute__((address_space(4))) int* trow;   // the request's table row: constant for the launch
    const char *kb, *vb;                                 // the pools at the key head, plus the lane's part of a tile
    uint32_t page_bytes;
    int n, i, g;
    bf16x8 qb[2]; f32x4 qf[4];   // Q^T operand: the one of T is used
    f32x4 c0[2];                 // slope * (row inside the lane's 8) in units of the score product
    float c1, slope2;
    float ref;                   // log2 reference of the probabilities; -inf: nothing seen yet
    f32x4 l, o[4];               // l: sum of the probabilities (bf16: in every register; fp32: the lane's own, register 0); o[j][r]: dimension 16 g + 4 r + j

    __device__ __forceinline__ Walk(const PagedAttnArgs& a_, int lane) : a(a_), i(lane & 15), g(lane >> 4) {}

    __device__ __forceinline__ void begin(int r, int n_, int kh, int head0, int heads) {
        n = n_;
        trow = (const __attribute__((address_space(4))) int*)(a.table + r * a.ld);
        page_bytes = (uint32_t)(a.kvh * HEAD * (int)sizeof(T)) << a.shift;
        const int mask = (1 << a.shift) - 1;
        kb = (const char*)((const T*)a.kp + row_offset(0, kh, (((i >> 2) * 8) & mask) + (i & 3), a.kvh, a.shift) + g * (sizeof(T) == 2 ? 8 : 4));
        vb = (const char*)((const T*)a.vp + row_offset(0, kh, (g * 8) & mask, a.kvh, a.shift) + i * 4);
        const bool on = i < heads;                  // columns behind the heads compute on zeros and are dropped
        const bool none = fabsf(a.scale) < 1e-20f;  // scores of nothing: q counts as 0 (the bias is divided by the scale)
        const T* q = (const T*)a.q + r * a.q_rs + (long)(head0 + (on ? i : 0)) * a.q_hs;   // any alignment: element loads
        const bool use = on && !none;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = q[32 * s + 8 * g + 2 * e], hi = q[32 * s + 8 * g + 2 * e + 1];
                    w[e] = use ? lo | hi << 16 : 0u;
                }
                qb[s] = __builtin_bit_cast(bf16x8, uint4{w[0], w[1], w[2], w[3]});
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
        for (int e = 0; e < 8; ++e) c0[e >> 2][e & 3] = per * (float)e;
        ref = -__builtin_inff(); l = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // rows outside the request count as its first or last one: their loads stay on its pages, their scores are dropped
    __device__ __forceinline__ Pages pages(int t) const {
        const uint32_t at = (uint32_t)max(t, 0) * TILE, last = (uint32_t)(n - 1) >> a.shift;
        Pages p;
#pragma unroll
        for (int c = 0; c < 4; ++c) p.id[c] = trow[min((at + 8 * c) >> a.shift, last)];
        return p;
    }
    // an entry that is no page: page 0's rows, masked by `ok`
    __device__ __forceinline__ void check(Pages& p) const {
#pragma unroll
        for (int c = 0; c < 4; ++c) { p.ok[c] = page_ok(p.id[c], a.num_pages); p.id[c] = p.ok[c] ? p.id[c] : 0; }
    }
    template <typename V> static __device__ __forceinline__ V of_group(const V (&v)[4], int c) { return c == 0 ? v[0] : c == 1 ? v[1] : c == 2 ? v[2] : v[3]; }

    template <bool NT> __device__ __forceinline__ void load_k(X& x, int t, const Pages& p) const {
        const uint32_t row = ((uint32_t)t * TILE & ((1u << a.shift) - 1u)) * (HEAD * sizeof(T));
        const char* k = kb + row + (uint64_t)(uint32_t)of_group(p.id, i >> 2) * page_bytes;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int s = 0; s < X::PER; ++s) {
                const auto* f = reinterpret_cast<const typename X::K*>(k + (tt * 4 * HEAD + s * (HEAD / X::PER)) * sizeof(T));
                x.k[tt][s] = NT ? __builtin_nontemporal_load(f) : *f;
            }
    }
    template <bool NT> __device__ __forceinline__ void load_v(X& x, int t, const Pages& p) const {
        const uint32_t row = ((uint32_t)t * TILE & ((1u << a.shift) - 1u)) * (HEAD * sizeof(T));
        const char* v = vb + row + (uint64_t)(uint32_t)of_group(p.id, g) * page_bytes;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const auto* f = reinterpret_cast<const typename X::V*>(v + e * HEAD * sizeof(T));
            x.v[e] = NT ? __builtin_nontemporal_load(f) : *f;
        }
    }

    __device__ __forceinline__ void scores(const X& x, f32x4 (&s)[2]) const {
        s[0] = c0[0]; s[1] = c0[1];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int e = 0; e < 2; ++e) s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.k[tt][e]), qb[e], s[tt], 0, 0, 0);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int f = 0; f < 4; ++f) s[tt] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[tt][e][f], qf[e][f], s[tt], 0, 0, 0);
            }
        }
    }

    __device__ __forceinline__ void weigh(X& x, const f32x4 (&s)[2], int t, const Pages& pg) {
        const int row0 = t * TILE + g * 8;
        const bool unset = ref == -__builtin_inff();
        const float base = __builtin_fmaf(slope2, (float)(row0 - (n - 1)), unset ? 0.f : -ref);
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = __builtin_fmaf(c1, s[e >> 2][e & 3], base);
        if (t * TILE + TILE > n || !(pg.ok[0] && pg.ok[1] && pg.ok[2] && pg.ok[3])) {   // rows behind the length or on no page: no weight, and no bit of theirs in the product
            const bool ok = of_group(pg.ok, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = ok && row0 + e < n;
                p[e] = in ? p[e] : -__builtin_inff();
#pragma unroll
                for (int f = 0; f < (int)(sizeof(x.v[0]) / 4); ++f) x.v[e][f] = in ? x.v[e][f] : 0;
            }
        }
        const float own = max3(max3(p[0], p[1], p[2]), max3(p[3], p[4], p[5]), max3(p[6], p[7], p[7]));
        if (__any(own > (unset ? -__builtin_inff() : RISE))) {   // rare: the walk goes from the newest rows, where the bias is largest, to the oldest
            const float up = quad_max(own);
            if (up > (unset ? -__builtin_inff() : RISE)) {
                const float c = unset ? 0.f : __builtin_amdgcn_exp2f(-up);   // (unset: nothing but zeros to scale)
                ref = unset ? up : ref + up;
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] -= up;
                l *= c;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] *= c;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(p[e]);
        if constexpr (sizeof(T) == 2) {
            u32x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t h = pack_bf2(p[2 * e], p[2 * e + 1]);
                asm("" : "+v"(h));   // (the low half by a shift of the pair, not by a second conversion)
                hi[e] = h;
                lo[e] = pack_bf2(p[2 * e] - __uint_as_float(h << 16), p[2 * e + 1] - __uint_as_float(h & 0xffff0000u));
            }
            const bf16x8 ph = __builtin_bit_cast(bf16x8, hi), pl = __builtin_bit_cast(bf16x8, lo);
            const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
            l = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, ph, l, 0, 0, 0);
            l = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pl, l, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_perm(x.v[2 * e + 1][j >> 1], x.v[2 * e][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
                const bf16x8 vt = __builtin_bit_cast(bf16x8, w);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, ph, o[j], 0, 0, 0);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, pl, o[j], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                l[0] += p[e];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[e][j], p[e], o[j], 0, 0, 0);
            }
        }
    }

    __device__ __forceinline__ float sum() const { return sizeof(T) == 2 ? l[0] : quad_sum(l[0]); }

    // Tiles t, t - WAVES, ... down to t0.  One tile's registers: the next tile's K replaces this one's as soon as its products are done, V the
    // same behind the second product, and the page ids come a tile earlier.
    template <bool NT> __device__ __forceinline__ void run(int t, int t0) {
        if (t < t0) return;
        X x;
        Pages now = pages(t), next = pages(t - WAVES);
        check(now);
        load_k<NT>(x, t, now);
        load_v<NT>(x, t, now);
        for (;;) {
            f32x4 s[2];
            scores(x, s);
            const bool more = t - WAVES >= t0;
            check(next);
            if (more) load_k<NT>(x, t - WAVES, next);
            const Pages then = pages(t - 2 * WAVES);
            weigh(x, s, t, now);
            if (!more) return;
            t -= WAVES;
            load_v<NT>(x, t, next);
            now = next; next = then;
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

// Inclusive sum over the wave's lanes (row shifts by 1, 2, 4, 8, then the rows' last lanes into the rows behind).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}

__device__ __forceinline__ int tiles_of(const PagedAttnArgs& a, int r) { return (rows_of(a.lens[r], a.W, a.shift) + TILE - 1) / TILE; }

// parts of a (request, key head, pass) of `tiles` tiles, none above `most` tiles unless there would be more than MAX_PARTS
constexpr int MAX_PARTS = 256;
__device__ __forceinline__ int parts_of(int tiles, int most) { return max(1, min(MAX_PARTS, (int)(((uint32_t)tiles + (uint32_t)most - 1u) / (uint32_t)most))); }

// One workgroup, one part of one (request, key head, pass).  DIRECT: the whole of it.  Otherwise every wave adds up the batch's tiles for
// itself (a lane: every 64th stretch of requests; no barrier, no LDS), takes a `target`-th of them as the longest part, and finds the
// request whose parts workgroup number wg is among.
template <typename T, bool DIRECT>
__global__ __launch_bounds__(64 * WAVES, sizeof(T) == 2 ? 4 : 3) void paged_attn_kernel(PagedAttnArgs a) {
    __shared__ float s_o[WAVES][HEADS][LDO], s_m[WAVES][HEADS], s_l[WAVES][HEADS];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), H = a.kvh * a.passes;
    const int wg = blockIdx.x;
    int r, hp, part = 0, parts = 1;
    if constexpr (DIRECT) {
        r = wg / H; hp = wg - r * H;
    } else {
        const int per = (a.R + 63) / 64, q0 = min(a.R, lane * per), q1 = min(a.R, q0 + per);   // this lane's requests
        const int c0 = q0 < q1 ? tiles_of(a, q0) : 0;
        long mine = c0;
        for (int q = q0 + 1; q < q1; ++q) mine += tiles_of(a, q);
        // in two halves of 32 bits: table capacities pass 2^32 tiles before memory does
        const long total = ((long)__builtin_amdgcn_readlane(wave_scan((int)(mine >> 16)), 63) << 16) + (uint32_t)__builtin_amdgcn_readlane(wave_scan((int)(mine & 0xffff)), 63);
        const int most = (int)min(max((long)MIN_TILES, (total * H + TARGET - 1) / TARGET), (long)a.max_tiles);
        int units = q0 < q1 ? H * parts_of(c0, most) : 0;
        for (int q = q0 + 1; q < q1; ++q) units += H * parts_of(tiles_of(a, q), most);
        const int incl = wave_scan(units);
        const unsigned long long behind = __ballot(incl > wg);
        if (!behind) {
            if (tid == 0) a.hdr[wg] = int4{0, 0, 0, 0};
            return;
        }
        const int at = __builtin_ctzll(behind);
        int off = wg - __builtin_amdgcn_readlane(incl - units, at);
        r = at * per;
        for (;;) {
            parts = parts_of(tiles_of(a, r), most);
            if (off < H * parts) break;
            off -= H * parts; ++r;
        }
        hp = off / parts; part = off - hp * parts;
    }
    r = __builtin_amdgcn_readfirstlane(r);
    const int n = rows_of(a.lens[r], a.W, a.shift), tiles = (n + TILE - 1) / TILE;
    const int t0 = DIRECT ? 0 : (int)((long)tiles * part / parts), t1 = DIRECT ? tiles : (int)((long)tiles * (part + 1) / parts);
    const int kh = hp / a.passes, first = (hp - kh * a.passes) * HEADS, heads = min(HEADS, a.group - first), head0 = kh * a.group + first;
    Walk<T> wk(a, lane);
    wk.begin(r, n, kh, head0, heads);
    if (a.once) wk.template run<true>(t1 - 1 - w, t0); else wk.template run<false>(t1 - 1 - w, t0);
    const float l = wk.sum();
    if (wk.g == 0) { s_m[w][wk.i] = wk.ref; s_l[w][wk.i] = l; }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(&s_o[w][wk.i][16 * wk.g + 4 * q]) = f32x4{wk.o[0][q], wk.o[1][q], wk.o[2][q], wk.o[3][q]};
    __syncthreads();
    const int hd = tid >> 4, d = (tid & 15) * 4;   // the first 256 threads: 16 heads x 16 pieces of 4 dimensions
    if (hd < heads) {
        float M = -__builtin_inff(), L = 0.f, O[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < WAVES; ++u) M = fmaxf(M, s_m[u][hd]);
#pragma unroll
        for (int u = 0; u < WAVES; ++u) {
            const float mu = s_m[u][hd], c = mu == -__builtin_inff() ? 0.f : mu == M ? 1.f : __builtin_amdgcn_exp2f(mu - M);
            const f32x4 ov = *reinterpret_cast<const f32x4*>(&s_o[u][hd][d]);
            L += c * s_l[u][hd];
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] += c * ov[e];
        }
        if (DIRECT || parts == 1) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] = L == 0.f ? 0.f : O[e] * inv;
            store4((T*)a.o + r * a.o_rs + (long)(head0 + hd) * a.o_hs + d, O);
        } else {
            const long slot = (long)wg * a.rows + hd;
            *reinterpret_cast<f32x4*>(a.part + slot * HEAD + d) = f32x4{O[0], O[1], O[2], O[3]};
            if (d == 0) { a.ml[2 * slot] = M; a.ml[2 * slot + 1] = L; }
        }
    }
    if (!DIRECT && tid == 0) a.hdr[wg] = int4{r, hp, part == 0 && parts > 1 ? parts : 0, 0};
}

// Joins the parts of a (request, key head, pass) that was cut: slots g .. g + parts - 1, in a fixed order.  JOIN_HEADS heads a block; 16 lanes
// (4 dimensions each) take every 8th part of a head, eight of them in flight.
constexpr int JOIN_HEADS = 2, JOIN_SUBS = 16 / JOIN_HEADS;
template <typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
    __shared__ float s_o[16][LDO], s_m[16], s_l[16];
    const long wg = blockIdx.x;
    const int4 cut = a.hdr[wg];
    if (cut.z == 0) return;
    const int kh = cut.y / a.passes, first = (cut.y - kh * a.passes) * HEADS, heads = min(HEADS, a.group - first), head0 = kh * a.group + first;
    const int grp = threadIdx.x >> 4, d = (threadIdx.x & 15) * 4, sub = grp % JOIN_SUBS, hd = blockIdx.y * JOIN_HEADS + grp / JOIN_SUBS;
    float M = -__builtin_inff(), L = 0.f;
    f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
    if (hd < heads) {
        const float* ml = a.ml + 2 * (wg * a.rows + hd);
        const float* po = a.part + (wg * a.rows + hd) * HEAD + d;
        constexpr int U = 8;
        for (int p = sub; p < cut.z; p += JOIN_SUBS * U) {
            float m[U], l[U];
            f32x4 o[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long at = (long)min(p + u * JOIN_SUBS, cut.z - 1) * a.rows;
                m[u] = ml[2 * at]; l[u] = ml[2 * at + 1];
                o[u] = *reinterpret_cast<const f32x4*>(po + at * HEAD);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (p + u * JOIN_SUBS >= cut.z) m[u] = -__builtin_inff(), l[u] = 0.f, o[u] = f32x4{0.f, 0.f, 0.f, 0.f};
                const float mn = fmaxf(M, m[u]), c = M == mn ? 1.f : __builtin_amdgcn_exp2f(M - mn);
                const float b = m[u] == -__builtin_inff() ? 0.f : m[u] == mn ? 1.f : __builtin_amdgcn_exp2f(m[u] - mn);
                L = L * c + l[u] * b; M = mn;
#pragma unroll
                for (int e = 0; e < 4; ++e) O[e] = O[e] * c + o[u][e] * b;
            }
        }
    }
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
            const float mu = s_m[grp + u], c = mu == -__builtin_inff() ? 0.f : mu == M ? 1.f : __builtin_amdgcn_exp2f(mu - M);
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

// Whether a workgroup takes a whole (request, key head, pass): one launch instead of two.  A lone workgroup reads 49 GB/s, the machine 4.9 TB/s,
// and the cut costs about 8 us (the count in front, the join behind it), so with rows enough to fill half of every table
//   cap / 49 GB/s  <=  segments * cap / 2 / 4.9 TB/s + 8 us,
// and never where one full table among short ones would take more than 21 us by itself (1 MiB: 4096 rows of a bf16 key head).
bool whole(long segments, long cap_bytes) {
#ifdef PA_DIRECT
    return PA_DIRECT;
#endif
    return cap_bytes <= (1L << 19) && cap_bytes * (200 - segments) <= 200L * 8 * 49000;
}

struct Split { long grid; bool direct; int passes, rows, max_tiles; };
Split split_of(int R, int h, int kvh, int W, int shift, int esize) {
    Split s;
    const int group = h / kvh;
    s.passes = (group + HEADS - 1) / HEADS; s.rows = group < HEADS ? group : HEADS;
    const long H = (long)kvh * s.passes, cap = (long)W << shift, tiles = (cap + TILE - 1) / TILE;
    s.direct = whole(R * H, cap * HEAD * 2 * esize);
    // the longest part: MAX_TILES, or what keeps the grid -- all tables full -- to 8192 parts
    const long full = R * H * tiles, most = (full + 8191) / 8192;
    s.max_tiles = (int)(most < MAX_TILES ? MAX_TILES : most);
    // parts on the device: tiles / most + 1 for each segment, with most >= MIN_TILES and most >= min(max_tiles, tiles / TARGET)
    long units = full / s.max_tiles + R * H;
    if (units < TARGET + R * H) units = TARGET + R * H;
    const long finest = R * H * ((tiles + MIN_TILES - 1) / MIN_TILES);
    s.grid = s.direct ? R * H : units < finest ? units : finest;
    return s;
}

int page_shift(int page) {
    for (int s = 3; s <= 12; ++s) if (page == 1 << s) return s;
    return -1;
}

size_t scratch_of(const Split& s) { return s.direct ? 0 : (size_t)s.grid * ((size_t)s.rows * (HEAD + 2) * sizeof(float) + sizeof(int4)); }

template <typename T, bool DIRECT>
int launch(const PagedAttnArgs& a, long grid, hipStream_t stream) {
    hipLaunchKernelGGL((paged_attn_kernel<T, DIRECT>), dim3((unsigned)grid), dim3(64 * WAVES), 0, stream, a);
    SPN_LAUNCH_CHECK();
    if (!DIRECT) {
        hipLaunchKernelGGL(paged_join_kernel<T>, dim3((unsigned)grid, cdiv(a.rows, JOIN_HEADS)), dim3(256), 0, stream, a);
        SPN_LAUNCH_CHECK();
    }
    return SPN_OK;
}

}  // namespace

extern "C" size_t spn_paged_attn_workspace_bytes(int R, int h, int kvh, int W, int page, int dtype) {
    const int shift = page_shift(page);
    if (shift < 0 || R < 1 || h < 1 || kvh < 1 || h % kvh || W < 1) return 0;   // refused by the call itself
    return scratch_of(split_of(R, h, kvh, W, shift, dtype == 1 ? 2 : 4));
}

extern "C" int spn_paged_attn(const void* q, long q_rs, long q_hs, const void* k_pages, const void* v_pages, int dtype, const int* block_table, long bt_ld,
                              const int* lens, const float* slopes, void* o, long o_rs, long o_hs, int R, int h, int kvh, int W, int num_pages,
                              int page, float scale, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const int shift = page_shift(page);
    SPN_REQUIRE(q && k_pages && v_pages && block_table && lens && o, "spn_paged_attn: null buffer");
    SPN_REQUIRE(dtype == 0 || dtype == 1, "spn_paged_attn: dtype codes are 0 (fp32) and 1 (bf16)");
    SPN_REQUIRE(shift >= 0, "spn_paged_attn: the page size must be a power of two in [8, 4096]");
    SPN_REQUIRE(R > 0 && h > 0 && kvh > 0 && h % kvh == 0 && W > 0 && num_pages > 0 && bt_ld >= W && ((long)W << shift) < (1L << 31) && (long)R * W < (1L << 31) &&
                (long)R * h < (1L << 21) &&
                ((long)kvh * HEAD * 4 << shift) < (1L << 32), "spn_paged_attn: bad sizes");
    SPN_REQUIRE(((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) == 0, "spn_paged_attn: pages must be 16-byte aligned");
    const Split s = split_of(R, h, kvh, W, shift, dtype == 1 ? 2 : 4);
    const size_t need = scratch_of(s);
    SPN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                "spn_paged_attn: the workspace is too small or not 16-byte aligned (spn_paged_attn_workspace_bytes)");
    PagedAttnArgs a{q, q_rs, q_hs, k_pages, v_pages, block_table, bt_ld, lens, slopes, o, o_rs, o_hs, R, h, kvh, W, num_pages, shift, scale,
                    h / kvh, s.passes, s.rows, s.max_tiles, 0, nullptr, nullptr, nullptr};
    if (!s.direct) {
        a.hdr = (int4*)workspace; a.part = (float*)(a.hdr + s.grid); a.ml = a.part + s.grid * s.rows * HEAD;
    }
    if (dtype == 1) return s.direct ? launch<bf16_t, true>(a, s.grid, stream) : launch<bf16_t, false>(a, s.grid, stream);
    return s.direct ? launch<float, true>(a, s.grid, stream) : launch<float, false>(a, s.grid, stream);
}
