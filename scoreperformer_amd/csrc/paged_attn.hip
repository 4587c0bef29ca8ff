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
constexpr int HEADS = 16;      // query heads per pass
constexpr int LDO = 68;        // LDS row of a head's o: 64 + 4, so that 16 heads do not meet in one bank
constexpr float LOG2E_F = 1.4426950408889634f;

struct PagedAttnArgs {
    const void* q; long q_rs, q_hs; const void* kp; const void* vp; const int* table; long ld; const int* lens; const float* slopes;
    void* o; long o_rs, o_hs; int R, h, kvh, W, num_pages, shift; float scale;
    int group, passes;         // query heads per key head, 16-head passes over them
    int rows;                  // heads of a partial result: min(group, 16)
    int min_tiles;             // least tiles of a workgroup
    float* part; float* ml; int4* hdr;   // [G][2][rows][64], [G][2][rows][2], [G]
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

// A tile's rows as they arrive.  Lane (i = lane & 15, g = lane >> 4).  K: tile row (i >> 2) * 8 + 4 t + (i & 3) for t = 0, 1, so that the C
// registers of the two products hold rows g * 8 .. g * 8 + 7.  V: rows g * 8 + 0 .. 7, dimensions 4 i .. 4 i + 3.
template <typename T> struct Tile;
template <> struct Tile<bf16_t> { typedef uint4 K; typedef uint2 V; static constexpr int PER = 2; K k[2][2]; V v[8]; bool ok; };   // k[t][s]: dimensions 32 s + 8 g ..
template <> struct Tile<float> { typedef f32x4 K; typedef f32x4 V; static constexpr int PER = 4; K k[2][4]; V v[8]; bool ok; };    // k[t][s]: dimensions 16 s + 4 g ..

struct PageIds { int k, v; };

// One wave's walk over some tiles of one (request, key head): the state of the softmax of 16 heads, a head per lane & 15.
template <typename T>
struct Walk {
    typedef Tile<T> X;
    const PagedAttnArgs& a;
    const int* trow; const T* kp; const T* vp;   // the request's table row; the pools at the key head, plus the lane's part of a row
    int n, i, g;
    bf16x8 qb[2]; f32x4 qf[4];   // Q^T operand: the one of T is used
    float c1, slope2;
    float m, l; f32x4 o[4];      // o[j][r]: dimension 16 g + 4 r + j

    __device__ __forceinline__ Walk(const PagedAttnArgs& a_, int lane) : a(a_), i(lane & 15), g(lane >> 4) {}

    __device__ __forceinline__ void begin(int r, int n_, int kh, int head0, int heads) {
        n = n_;
        trow = a.table + r * a.ld;
        kp = (const T*)a.kp + row_offset(0, kh, i & 3, a.kvh, a.shift) + g * (sizeof(T) == 2 ? 8 : 4);
        vp = (const T*)a.vp + row_offset(0, kh, 0, a.kvh, a.shift) + i * 4;
        const bool on = i < heads;   // columns behind the heads compute on zeros and are dropped
        const T* q = (const T*)a.q + r * a.q_rs + (long)(head0 + (on ? i : 0)) * a.q_hs;   // any alignment: element loads
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = q[32 * s + 8 * g + 2 * e], hi = q[32 * s + 8 * g + 2 * e + 1];
                    w[e] = on ? lo | hi << 16 : 0u;
                }
                qb[s] = __builtin_bit_cast(bf16x8, uint4{w[0], w[1], w[2], w[3]});
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) { const float x = q[16 * s + 4 * g + e]; qf[s][e] = on ? x : 0.f; }
        }
        c1 = a.scale * LOG2E_F;
        slope2 = a.slopes ? a.slopes[head0 + (on ? i : 0)] * LOG2E_F : 0.f;
        m = -__builtin_inff(); l = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // page ids of tile t's rows; rows outside the request count as its first or last one (their loads stay on its pages, their scores are dropped)
    __device__ __forceinline__ PageIds pages(int t) const {
        const int at = max(t, 0) * TILE;
        return PageIds{trow[min(at + (i >> 2) * 8, n - 1) >> a.shift], trow[min(at + g * 8, n - 1) >> a.shift]};
    }

    // an entry that is no page: page 0's rows, masked by `ok`
    __device__ __forceinline__ void load_k(X& x, int t, const PageIds id) const {
        const T* k = kp + row_offset(page_ok(id.k, a.num_pages) ? id.k : 0, 0, (t * TILE + (i >> 2) * 8) & ((1 << a.shift) - 1), a.kvh, a.shift);
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int s = 0; s < X::PER; ++s) x.k[tt][s] = *reinterpret_cast<const typename X::K*>(k + tt * 4 * HEAD + s * (HEAD / X::PER));
    }
    __device__ __forceinline__ void load_v(X& x, int t, const PageIds id) const {
        x.ok = page_ok(id.v, a.num_pages);
        const T* v = vp + row_offset(x.ok ? id.v : 0, 0, (t * TILE + g * 8) & ((1 << a.shift) - 1), a.kvh, a.shift);
#pragma unroll
        for (int e = 0; e < 8; ++e) x.v[e] = *reinterpret_cast<const typename X::V*>(v + e * HEAD);
    }

    __device__ __forceinline__ void scores(const X& x, f32x4 (&s)[2]) const {
        s[0] = f32x4{0.f, 0.f, 0.f, 0.f}; s[1] = s[0];
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

    __device__ __forceinline__ void weigh(X& x, const f32x4 (&s)[2], int t) {
        const int row0 = t * TILE + g * 8;
        const float base = slope2 * (float)(row0 - (n - 1));
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = __builtin_fmaf(c1, s[e >> 2][e & 3], __builtin_fmaf(slope2, (float)e, base));
        if (!(t * TILE + TILE <= n && __all(x.ok))) {   // rows behind the length or on no page: no weight, and no bit of theirs in the product
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = x.ok && row0 + e < n;
                p[e] = in ? p[e] : -__builtin_inff();
                if constexpr (sizeof(T) == 2) { x.v[e].x = in ? x.v[e].x : 0u; x.v[e].y = in ? x.v[e].y : 0u; }
                else {
#pragma unroll
                    for (int f = 0; f < 4; ++f) x.v[e][f] = in ? x.v[e][f] : 0.f;
                }
            }
        }
        const float mx = quad_max(fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7]))));
        if (__any(mx > m)) {   // rare: the walk goes from the newest rows, where the bias is largest, to the oldest
            const float mn = fmaxf(m, mx), c = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn; l *= c;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] *= c;
        }
        const float ms = m == -__builtin_inff() ? 0.f : m;   // nothing visible so far: every p is exp2(-inf) = 0
#pragma unroll
        for (int e = 0; e < 8; ++e) { p[e] = __builtin_amdgcn_exp2f(p[e] - ms); l += p[e]; }
        if constexpr (sizeof(T) == 2) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi[e] = pack_bf2(p[2 * e], p[2 * e + 1]);
                lo[e] = pack_bf2(p[2 * e] - __uint_as_float(hi[e] << 16), p[2 * e + 1] - __uint_as_float(hi[e] & 0xffff0000u));
            }
            const bf16x8 ph = __builtin_bit_cast(bf16x8, uint4{hi[0], hi[1], hi[2], hi[3]}), pl = __builtin_bit_cast(bf16x8, uint4{lo[0], lo[1], lo[2], lo[3]});
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t v0 = j < 2 ? x.v[2 * e].x : x.v[2 * e].y, v1 = j < 2 ? x.v[2 * e + 1].x : x.v[2 * e + 1].y;
                    w[e] = __builtin_amdgcn_perm(v1, v0, j & 1 ? 0x07060302u : 0x05040100u);
                }
                const bf16x8 vt = __builtin_bit_cast(bf16x8, uint4{w[0], w[1], w[2], w[3]});
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, ph, o[j], 0, 0, 0);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, pl, o[j], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[e][j], p[e], o[j], 0, 0, 0);
        }
    }

    // Tiles t, t - STEP, ... down to t0.  One tile's registers: the next tile's K replaces this one's as soon as its products are done, V the
    // same behind the second product, and the page ids come a tile earlier.  Loads return in order, so they are issued in the order of their
    // use (K, ids, V) and every wait leaves the younger ones in flight.
    template <int STEP>
    __device__ __forceinline__ void run(int t, int t0) {
        if (t < t0) return;
        X x;
        PageIds id = pages(t);
        load_k(x, t, id);
        PageIds next = pages(t - STEP);
        load_v(x, t, id);
        for (;;) {
            f32x4 s[2];
            scores(x, s);
            const bool more = t - STEP >= t0;
            id = next;
            if (more) load_k(x, t - STEP, id);
            next = pages(t - 2 * STEP);
            weigh(x, s, t);
            if (!more) return;
            t -= STEP;
            load_v(x, t, id);
        }
    }
};

__device__ __forceinline__ long uniform(long v) {
    return (long)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

template <typename T>
__device__ __forceinline__ void store4(T* to, const float (&v)[4]) {   // any alignment
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 2) to[e] = f2bf(v[e]); else to[e] = v[e];
    }
}

// DIRECT: workgroup = one (request, key head, pass), no cut.  Otherwise the G-th part of the line of tiles.
template <typename T, bool DIRECT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, sizeof(T) == 2 ? 4 : 3) void paged_attn_kernel(PagedAttnArgs a) {
    __shared__ float s_o[WAVES][HEADS][LDO], s_m[WAVES][HEADS], s_l[WAVES][HEADS];
    __shared__ long s_sum[WAVES], s_at[3];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), H = a.kvh * a.passes;
    const long wg = blockIdx.x;
    long lo = 0, hi = 0, N = 0, G = 1, base = 0;
    int r;
    if constexpr (DIRECT) {
        r = (int)(wg / H);
    } else {
        // requests without a row: zeros
        for (int q = (int)wg; q < a.R; q += gridDim.x)
            if (rows_of(a.lens[q], a.W, a.shift) == 0)
                for (int e = tid; e < a.h * HEAD; e += 64 * WAVES) ((T*)a.o)[q * a.o_rs + (long)(e / HEAD) * a.o_hs + e % HEAD] = 0;
        // the line of tiles: a thread sums up `per` requests, the block the threads
        const int per = (a.R + 64 * WAVES - 1) / (64 * WAVES), q0 = min(a.R, tid * per), q1 = min(a.R, q0 + per);
        long mine = 0;
        for (int q = q0; q < q1; ++q) mine += (rows_of(a.lens[q], a.W, a.shift) + TILE - 1) / TILE;
        long incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const long u = __shfl_up(incl, d, 64);
            if (lane >= d) incl += u;
        }
        if (lane == 63) s_sum[w] = incl;
        __syncthreads();
        long before = 0;
#pragma unroll
        for (int u = 0; u < WAVES; ++u) { before += u < w ? s_sum[u] : 0; N += s_sum[u]; }
        incl += before;
        N = uniform(N * H);
        G = min((long)gridDim.x, max(1L, (N + a.min_tiles - 1) / a.min_tiles));
        lo = wg < G ? wg * N / G : 0; hi = wg < G ? (wg + 1) * N / G : 0;
        if (lo < hi && (incl - mine) * H <= lo && lo < incl * H) {   // exactly one thread: find the request
            long at = (incl - mine) * H;
            int q = q0;
            for (;; ++q) {
                const long c = (long)((rows_of(a.lens[q], a.W, a.shift) + TILE - 1) / TILE) * H;
                if (lo < at + c) break;
                at += c;
            }
            s_at[0] = q; s_at[1] = at;
        }
        __syncthreads();
        if (lo >= hi) {
            if (tid == 0) a.hdr[wg] = int4{-1, 0, 0, 0};
            return;
        }
        r = (int)s_at[0]; base = uniform(s_at[1]);
    }
    r = __builtin_amdgcn_readfirstlane(r);
    int4 cut = int4{-1, 0, 0, 0};
    Walk<T> wk(a, lane);
    for (long at = lo;;) {
        const int n = rows_of(a.lens[r], a.W, a.shift), tiles = (n + TILE - 1) / TILE;
        if (!DIRECT && tiles == 0) {
            if (++r >= a.R) break;   // (never: the line has tiles up to hi)
            continue;
        }
        int hp, t0, t1;
        if constexpr (DIRECT) { hp = (int)(wg - (long)r * H); t0 = 0; t1 = tiles; }
        else {
            const long off = at - base;
            hp = (int)(off / tiles);
            t0 = (int)(off - (long)hp * tiles);
            t1 = (int)min((long)tiles, t0 + (hi - at));
        }
        const int kh = hp / a.passes, first = (hp - kh * a.passes) * HEADS, heads = min(HEADS, a.group - first), head0 = kh * a.group + first;
        wk.begin(r, n, kh, head0, heads);
        wk.template run<WAVES>(t1 - 1 - w, t0);
        const float l = quad_sum(wk.l);
        if (wk.g == 0) { s_m[w][wk.i] = wk.m; s_l[w][wk.i] = l; }
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
            if (DIRECT || (t0 == 0 && t1 == tiles)) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
                for (int e = 0; e < 4; ++e) O[e] = L == 0.f ? 0.f : O[e] * inv;
                store4((T*)a.o + r * a.o_rs + (long)(head0 + hd) * a.o_hs + d, O);
            } else {
                const long slot = ((2 * wg + (t0 == 0)) * a.rows + hd);
                *reinterpret_cast<f32x4*>(a.part + slot * HEAD + d) = f32x4{O[0], O[1], O[2], O[3]};
                if (d == 0) { a.ml[2 * slot] = M; a.ml[2 * slot + 1] = L; }
            }
        }
        if constexpr (DIRECT) return;
        if (t0 == 0 && t1 < tiles)   // begins here, goes on behind: this workgroup's entry names the last one that has a part of it
            cut = int4{r, hp, (int)(((base + (long)(hp + 1) * tiles) * G - 1) / N), 0};
        at += t1 - t0;
        if (at >= hi) break;
        if (at == base + (long)tiles * H) { base = at; if (++r >= a.R) break; }
        __syncthreads();
    }
    if (tid == 0) a.hdr[wg] = cut;
}

// Joins a request that was cut: workgroup g's second partial, then the first partials of g + 1 .. last, in this order.
constexpr int JOIN = 4;   // parts of the list, a quarter of the block each
template <typename T>
__global__ __launch_bounds__(256 * JOIN) void paged_join_kernel(PagedAttnArgs a) {
    __shared__ float s_o[JOIN][HEADS][LDO], s_m[JOIN][HEADS], s_l[JOIN][HEADS];
    const int4 cut = a.hdr[blockIdx.x];
    if (cut.x < 0) return;
    const long wg = blockIdx.x;
    const int kh = cut.y / a.passes, first = (cut.y - kh * a.passes) * HEADS, heads = min(HEADS, a.group - first), head0 = kh * a.group + first;
    const int sub = threadIdx.x >> 8, hd = (threadIdx.x >> 4) & 15, d = (threadIdx.x & 15) * 4, np = cut.z - (int)wg + 1;
    float M = -__builtin_inff(), L = 0.f;
    f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
    if (hd < heads) {
        for (int p = sub; p < np; p += JOIN) {
            const long slot = ((2 * (wg + p) + (p == 0)) * a.rows + hd);
            const float m = a.ml[2 * slot], l = a.ml[2 * slot + 1];
            const f32x4 o = *reinterpret_cast<const f32x4*>(a.part + slot * HEAD + d);
            const float mn = fmaxf(M, m), c = M == mn ? 1.f : __builtin_amdgcn_exp2f(M - mn), b = m == -__builtin_inff() ? 0.f : m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            L = L * c + l * b; M = mn;
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] = O[e] * c + o[e] * b;
        }
        *reinterpret_cast<f32x4*>(&s_o[sub][hd][d]) = O;
        if (d == 0) { s_m[sub][hd] = M; s_l[sub][hd] = L; }
    }
    __syncthreads();
    if (sub == 0 && hd < heads) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        M = -__builtin_inff(); L = 0.f;
        for (int u = 0; u < JOIN; ++u) M = fmaxf(M, s_m[u][hd]);
        for (int u = 0; u < JOIN; ++u) {
            const float mu = s_m[u][hd], c = mu == -__builtin_inff() ? 0.f : mu == M ? 1.f : __builtin_amdgcn_exp2f(mu - M);
            L += c * s_l[u][hd];
            for (int e = 0; e < 4; ++e) v[e] += c * s_o[u][hd][d + e];
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        for (int e = 0; e < 4; ++e) v[e] = L == 0.f ? 0.f : v[e] * inv;
        store4((T*)a.o + cut.x * a.o_rs + (long)(head0 + hd) * a.o_hs + d, v);
    }
}

#ifndef PA_MIN_TILES
#define PA_MIN_TILES 8
#endif
#ifndef PA_DIRECT_ROWS
#define PA_DIRECT_ROWS 256
#endif
#ifndef PA_SPLIT_WAVES
#define PA_SPLIT_WAVES 4
#endif
#ifndef PA_DIRECT_WAVES
#define PA_DIRECT_WAVES 4
#endif
constexpr int MIN_TILES = PA_MIN_TILES;       // two tiles a wave
constexpr int DIRECT_ROWS = PA_DIRECT_ROWS;   // tables of at most this many rows: a workgroup per (request, key head)
constexpr int SPLIT_WAVES = PA_SPLIT_WAVES, DIRECT_WAVES = PA_DIRECT_WAVES;

struct Split { long grid; bool direct; int passes, rows; };
Split split_of(int R, int h, int kvh, int W, int shift, int esize) {
    Split s;
    const int group = h / kvh;
    s.passes = (group + HEADS - 1) / HEADS; s.rows = group < HEADS ? group : HEADS;
    const long H = (long)kvh * s.passes, cap = (long)W << shift, tiles = (cap + TILE - 1) / TILE;
    s.direct = cap <= DIRECT_ROWS;
    const long most = 256 * (esize == 2 ? 4 : 3) * 4 / SPLIT_WAVES, units = (tiles * H + MIN_TILES - 1) / MIN_TILES * R;
    s.grid = s.direct ? R * H : units < most ? units : most;
    return s;
}

int page_shift(int page) {
    for (int s = 3; s <= 12; ++s) if (page == 1 << s) return s;
    return -1;
}

size_t scratch_of(const Split& s) { return s.direct ? 0 : (size_t)s.grid * (2 * (size_t)s.rows * (HEAD + 2) * sizeof(float) + sizeof(int4)); }

template <typename T, bool DIRECT>
int launch(const PagedAttnArgs& a, long grid, hipStream_t stream) {
    constexpr int WAVES = DIRECT ? DIRECT_WAVES : SPLIT_WAVES;
    hipLaunchKernelGGL((paged_attn_kernel<T, DIRECT, WAVES>), dim3((unsigned)grid), dim3(64 * WAVES), 0, stream, a);
    SPN_LAUNCH_CHECK();
    if (!DIRECT) {
        hipLaunchKernelGGL(paged_join_kernel<T>, dim3((unsigned)grid), dim3(256 * JOIN), 0, stream, a);
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
                (long)R * h < (1L << 31), "spn_paged_attn: bad sizes");
    SPN_REQUIRE(((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) == 0, "spn_paged_attn: pages must be 16-byte aligned");
    const Split s = split_of(R, h, kvh, W, shift, dtype == 1 ? 2 : 4);
    const size_t need = scratch_of(s);
    SPN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                "spn_paged_attn: the workspace is too small or not 16-byte aligned (spn_paged_attn_workspace_bytes)");
    PagedAttnArgs a{q, q_rs, q_hs, k_pages, v_pages, block_table, bt_ld, lens, slopes, o, o_rs, o_hs, R, h, kvh, W, num_pages, shift, scale,
                    h / kvh, s.passes, s.rows, MIN_TILES, nullptr, nullptr, nullptr};
    if (!s.direct) {
        a.hdr = (int4*)workspace; a.part = (float*)(a.hdr + s.grid); a.ml = a.part + 2 * s.grid * s.rows * HEAD;
    }
    if (dtype == 1) return s.direct ? launch<bf16_t, true>(a, s.grid, stream) : launch<bf16_t, false>(a, s.grid, stream);
    return s.direct ? launch<float, true>(a, s.grid, stream) : launch<float, false>(a, s.grid, stream);
}
