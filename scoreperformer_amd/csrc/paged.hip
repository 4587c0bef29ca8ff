// The paged key / value cache (attention of a batch of requests whose lengths differ and grow): pages of 2^shift rows out of one pool,
// a block table [R, W] of page ids per request, the free pages a stack of ids in device memory.  Nothing here reads back to the host.
//   spn_paged_plan     lengths + new rows per request -> pages taken off the stack, block table, slot of every new row
//   spn_paged_release  pages of ended requests back on the stack
//   spn_paged_append   key / value rows -> their slots (converted on the way when the pool's type differs)
// The attention over the pages is paged_attn.hip.
#include "common.h"
#include "paged_index.h"

using namespace spn_paged;

namespace {

constexpr int PLAN_T = 1024;

// inclusive sum over the block's 1024 threads; `red`: 16 ints of LDS.  Two barriers, usable again after it returns.
__device__ __forceinline__ int block_scan(int v, int* red) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    if (lane == 63) red[w] = v;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < w; ++i) before += red[i];
    __syncthreads();
    return v + before;
}

struct PlanArgs {
    const int* lens; const int* fresh; int* table; long ld; const int* stack; const int* num_free; int* lens_out; int* num_free_out;
    long long* slots; int R, W, num_pages, shift, width;
    int4* rec;   // [R] {rows held, rows given, stack position of the first new page, 0}: what the second launch needs; null: one launch
};

// Slot i of request r: rows behind len + given and rows whose page id is no page get -1.  `top`: stack position of the request's first new
// page (its later ones lie below).  Every new page begins at exactly one new row, whose thread enters it into the table.
__device__ __forceinline__ void plan_emit(const PlanArgs& a, int r, int i, int len, int given, int top) {
    long slot = -1;
    if (i < given) {
        const long pos = (long)len + i;
        const int j = (int)(pos >> a.shift), held = (int)pages_of(len, a.shift);
        int id;
        if (j < held) id = a.table[r * a.ld + j];
        else {
            id = a.stack[top - (j - held)];
            if ((pos & ((1 << a.shift) - 1)) == 0) a.table[r * a.ld + j] = id;
        }
        slot = slot_of(id, pos, a.num_pages, a.shift);
    }
    a.slots[(long)r * a.width + i] = slot;
}

// One workgroup: the pages of request r lie behind those of the requests before it, an exclusive sum over the requests.  A request is
// served whole or not at all; once the pages asked for pass what is free, later requests that need one get none (the sum keeps growing),
// so the served ones take a contiguous piece off the top of the stack.  Latency is all there is: a decode step (one row per request) is
// lengths -> sum -> page id -> slot, four trips to memory, and is finished here (64 requests: 3.3 us); the slots of prompts are left to
// the whole machine (plan_fill_kernel).
template <bool FILL>
__global__ __launch_bounds__(PLAN_T) void plan_kernel(PlanArgs a) {
    __shared__ int red[16], s_len[PLAN_T], s_given[PLAN_T], s_top[PLAN_T], s_taken;
    const int tid = threadIdx.x;
    const int nf = min(max(*a.num_free, 0), a.num_pages);
    if (tid == 0) s_taken = 0;
    long carry = 0;
    for (int r0 = 0; r0 < a.R; r0 += PLAN_T) {
        const int r = r0 + tid, n = min(PLAN_T, a.R - r0);
        int len = 0, fresh = 0, need = -1;
        if (r < a.R) { len = a.lens[r]; fresh = a.fresh[r]; need = pages_needed(len, fresh, a.width, a.W, a.shift); }
        const int incl = block_scan(max(need, 0), red);
        const long end = carry + incl;
        const bool served = need >= 0 && (need == 0 || end <= nf);
        const int given = served ? fresh : 0, top = nf - 1 - (int)(end - max(need, 0));
        if (r < a.R) {
            a.lens_out[r] = served ? len + fresh : len;
            if (!FILL) a.rec[r] = int4{len, given, top, 0};
        }
        if (FILL) { s_len[tid] = len; s_given[tid] = given; s_top[tid] = top; }
        if (served && need > 0) atomicMax(&s_taken, (int)end);
        if (tid == PLAN_T - 1) red[0] = incl;
        __syncthreads();
        carry += red[0];
        if (FILL) {
#pragma unroll 4
            for (int e = tid; e < n * a.width; e += PLAN_T) {   // at most FILL_ONE
                const int q = e / a.width, i = e - q * a.width;
                plan_emit(a, r0 + q, i, s_len[q], s_given[q], s_top[q]);
            }
        }
        __syncthreads();
    }
    if (tid == 0) *a.num_free_out = nf - s_taken;
}

constexpr int FILL_ONE = 8192;   // slots up to which one workgroup fills them itself (64 x 128: 9.5 us; in two launches 8.3, and 4 us more of host time; 64 x 256: 13.7)
constexpr int FILL_B = 1024;     // slots of a workgroup of the second launch

__global__ __launch_bounds__(256) void plan_fill_kernel(PlanArgs a) {
    const uint32_t total = (uint32_t)a.R * (uint32_t)a.width;
#pragma unroll
    for (int u = 0; u < FILL_B / 256; ++u) {
        const uint32_t e = blockIdx.x * (uint32_t)FILL_B + u * 256u + threadIdx.x;
        if (e >= total) return;
        const uint32_t r = e / (uint32_t)a.width;
        const int4 c = a.rec[r];
        plan_emit(a, (int)r, (int)(e - r * (uint32_t)a.width), c.x, c.y, c.z);
    }
}

struct ReleaseArgs { const uint8_t* done; int* lens; int* table; long ld; int* stack; int* num_free; int R, W, num_pages, shift; int* cnt; };

// First of two launches, a wave per request: how many pages of the ended requests go back (cnt [R]); cnt[R]: the stack's height before.
__global__ __launch_bounds__(256) void release_count_kernel(ReleaseArgs a) {
    const int lane = threadIdx.x & 63, r = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.cnt[a.R] = min(max(*a.num_free, 0), a.num_pages);
    if (r >= a.R) return;
    int c = 0;
    if (a.done[r]) {
        const int held = (int)min(pages_of(a.lens[r], a.shift), (long)a.W);
        for (int j = lane; j < held; j += 64) c += page_ok(a.table[r * a.ld + j], a.num_pages);
#pragma unroll
        for (int d = 32; d; d >>= 1) c += __shfl_xor(c, d, 64);
    }
    if (lane == 0) a.cnt[r] = c;
}

// Second launch: 16 requests a workgroup, a wave each; every workgroup sums up the counts itself.  The pages go back so that page 0 of the
// first ended request lies on top of the stack: a plan for the same requests and lengths takes the same pages again.
__global__ __launch_bounds__(PLAN_T) void release_kernel(ReleaseArgs a) {
    __shared__ int red[16], s_before[16], s_total;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, first = blockIdx.x * 16;
    const int nf = a.cnt[a.R];
    int carry = 0;
    for (int r0 = 0; r0 < a.R; r0 += PLAN_T) {
        const int r = r0 + tid, mine = r < a.R ? a.cnt[r] : 0, incl = block_scan(mine, red);
        if (r >= first && r < first + 16) s_before[r - first] = carry + incl - mine;
        if (tid == PLAN_T - 1) s_total = incl;
        __syncthreads();
        carry += s_total;
        __syncthreads();
    }
    const int r = first + w;
    if (r < a.R && a.done[r]) {
        const int held = (int)min(pages_of(a.lens[r], a.shift), (long)a.W);
        long at = (long)nf + carry - 1 - s_before[w];
        for (int j = 0; j < held; j += 64) {
            const int id = j + lane < held ? a.table[r * a.ld + j + lane] : -1;
            const bool ok = page_ok(id, a.num_pages);
            const unsigned long long m = __ballot(ok);
            const long to = at - __popcll(m & ((1ull << lane) - 1));
            if (ok && to >= 0 && to < a.num_pages) a.stack[to] = id;      // past the end: more pages come back than the pool has, one was held twice
            if (j + lane < held) a.table[r * a.ld + j + lane] = -1;
            at -= __popcll(m);
        }
        if (lane == 0) a.lens[r] = 0;
    }
    if (blockIdx.x == 0 && tid == 0) *a.num_free = (int)min((long)nf + carry, (long)a.num_pages);
}

struct AppendArgs {
    const void* k; const void* v; long k_rs, k_hs, v_rs, v_hs; void* k_pages; void* v_pages; const long long* slots; long T; int kvh, num_pages, shift;
};

template <typename T> __device__ __forceinline__ float load1(const T* p) {
    if constexpr (sizeof(T) == 2) return bf2f(*p); else return *p;
}

// Any alignment: a thread moves one element of a key row and of the value row of the same note.
template <typename S, typename D>
__global__ __launch_bounds__(256) void append_any_kernel(AppendArgs a) {
    const long e = (long)blockIdx.x * 256 + threadIdx.x, row = e / (a.kvh * HEAD);
    if (row >= a.T) return;
    const int c = (int)(e - row * (a.kvh * HEAD)), head = c / HEAD, d = c % HEAD;
    const long slot = a.slots[row];
    if (!slot_ok(slot, a.num_pages, a.shift)) return;
    const long to = row_offset(slot >> a.shift, head, slot & ((1L << a.shift) - 1), a.kvh, a.shift) + d;
    const float k = load1((const S*)a.k + row * a.k_rs + head * a.k_hs + d), v = load1((const S*)a.v + row * a.v_rs + head * a.v_hs + d);
    if constexpr (sizeof(D) == 2) { ((D*)a.k_pages)[to] = f2bf(k); ((D*)a.v_pages)[to] = f2bf(v); }
    else { ((D*)a.k_pages)[to] = k; ((D*)a.v_pages)[to] = v; }
}

struct Eight { float x[8]; };
template <typename T> __device__ __forceinline__ Eight load8(const T* p) {
    Eight r;
    if constexpr (sizeof(T) == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) { r.x[2 * e] = __uint_as_float(w[e] << 16); r.x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
    } else {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { r.x[e] = lo[e]; r.x[4 + e] = hi[e]; }
    }
    return r;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Eight& r) {
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint4*>(p) = uint4{pack_bf2(r.x[0], r.x[1]), pack_bf2(r.x[2], r.x[3]), pack_bf2(r.x[4], r.x[5]), pack_bf2(r.x[6], r.x[7])};
    else {
        *reinterpret_cast<f32x4*>(p) = f32x4{r.x[0], r.x[1], r.x[2], r.x[3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{r.x[4], r.x[5], r.x[6], r.x[7]};
    }
}

// 16-byte aligned rows: a thread moves 8 elements of a key row and of the value row of the same note, 16-byte accesses throughout; 8 lanes
// fill one 128-byte line of a bf16 page.  Bound by HBM.
template <typename S, typename D>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    const uint32_t e = blockIdx.x * 256u + threadIdx.x, per = (uint32_t)a.kvh * 8, row = e / per;
    if (row >= a.T) return;
    const uint32_t c = e - row * per, head = c >> 3, d = (c & 7) * 8;
    const long slot = a.slots[row];
    const Eight k = load8((const S*)a.k + row * a.k_rs + head * a.k_hs + d), v = load8((const S*)a.v + row * a.v_rs + head * a.v_hs + d);
    if (!slot_ok(slot, a.num_pages, a.shift)) return;
    const long to = row_offset(slot >> a.shift, (int)head, slot & ((1L << a.shift) - 1), a.kvh, a.shift) + d;
    store8((D*)a.k_pages + to, k);
    store8((D*)a.v_pages + to, v);
}

template <typename S, typename D>
void append_launch(const AppendArgs& a, hipStream_t stream) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages) |
                           (uintptr_t)((a.k_rs | a.k_hs | a.v_rs | a.v_hs) * (long)sizeof(S));
    if (bits & 15) hipLaunchKernelGGL((append_any_kernel<S, D>), dim3(cdiv(a.T * a.kvh * HEAD, 256)), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((append_kernel<S, D>), dim3(cdiv(a.T * a.kvh * 8, 256)), dim3(256), 0, stream, a);
}

int log2_page(int page) {   // -1: not a power of two in [8, 4096]
    for (int s = 3; s <= 12; ++s) if (page == 1 << s) return s;
    return -1;
}

}  // namespace

extern "C" size_t spn_paged_plan_workspace_bytes(int R, int width) {
    return R > 0 && width > 0 && (long)R * width > FILL_ONE ? (size_t)R * sizeof(int4) : 0;
}

extern "C" int spn_paged_plan(const int* lens, const int* fresh, int* block_table, long bt_ld, const int* free_pages, const int* num_free,
                              int* lens_out, int* num_free_out, long long* slots, int R, int W, int num_pages, int page, int width,
                              void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const int shift = log2_page(page);
    SPN_REQUIRE(lens && fresh && block_table && free_pages && num_free && lens_out && num_free_out && slots, "spn_paged_plan: null buffer");
    SPN_REQUIRE(shift >= 0, "spn_paged_plan: the page size must be a power of two in [8, 4096]");
    SPN_REQUIRE(R > 0 && R < (1 << 24) && W > 0 && num_pages > 0 && width > 0 && bt_ld >= W, "spn_paged_plan: bad sizes");
    SPN_REQUIRE((long)R * W < (1L << 31) && ((long)W << shift) < (1L << 31) && (long)R * width < (1L << 31), "spn_paged_plan: sizes pass 2^31");
    const size_t need = spn_paged_plan_workspace_bytes(R, width);
    SPN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                "spn_paged_plan: the workspace is too small or not 16-byte aligned (spn_paged_plan_workspace_bytes)");
    const PlanArgs a{lens, fresh, block_table, bt_ld, free_pages, num_free, lens_out, num_free_out, slots, R, W, num_pages, shift, width, need ? (int4*)workspace : nullptr};
    if (need == 0) hipLaunchKernelGGL(plan_kernel<true>, dim3(1), dim3(PLAN_T), 0, stream, a);
    else {
        hipLaunchKernelGGL(plan_kernel<false>, dim3(1), dim3(PLAN_T), 0, stream, a);
        SPN_LAUNCH_CHECK();
        hipLaunchKernelGGL(plan_fill_kernel, dim3(cdiv((long)R * width, FILL_B)), dim3(256), 0, stream, a);
    }
    SPN_LAUNCH_CHECK();
    return SPN_OK;
}

extern "C" int spn_paged_release(const uint8_t* done, int* lens, int* block_table, long bt_ld, int* free_pages, int* num_free, int R, int W,
                                 int num_pages, int page, int* workspace, hipStream_t stream) {
    const int shift = log2_page(page);
    SPN_REQUIRE(done && lens && block_table && free_pages && num_free && workspace, "spn_paged_release: null buffer");
    SPN_REQUIRE(shift >= 0, "spn_paged_release: the page size must be a power of two in [8, 4096]");
    SPN_REQUIRE(R > 0 && R < (1 << 24) && W > 0 && num_pages > 0 && bt_ld >= W && (long)R * W < (1L << 31), "spn_paged_release: bad sizes");
    const ReleaseArgs a{done, lens, block_table, bt_ld, free_pages, num_free, R, W, num_pages, shift, workspace};
    hipLaunchKernelGGL(release_count_kernel, dim3(cdiv(R, 4)), dim3(256), 0, stream, a);
    SPN_LAUNCH_CHECK();
    hipLaunchKernelGGL(release_kernel, dim3(cdiv(R, 16)), dim3(PLAN_T), 0, stream, a);
    SPN_LAUNCH_CHECK();
    return SPN_OK;
}

extern "C" int spn_paged_append(const void* k, const void* v, int row_dtype, long k_rs, long k_hs, long v_rs, long v_hs, void* k_pages, void* v_pages,
                                int page_dtype, const long long* slots, long T, int kvh, int num_pages, int page, hipStream_t stream) {
    const int shift = log2_page(page);
    SPN_REQUIRE(k && v && k_pages && v_pages && slots, "spn_paged_append: null buffer");
    SPN_REQUIRE((row_dtype | page_dtype) >> 1 == 0, "spn_paged_append: dtype codes are 0 (fp32) and 1 (bf16)");
    SPN_REQUIRE(shift >= 0, "spn_paged_append: the page size must be a power of two in [8, 4096]");
    SPN_REQUIRE(T > 0 && kvh > 0 && num_pages > 0 && T * kvh < (1L << 26), "spn_paged_append: bad sizes");
    const AppendArgs a{k, v, k_rs, k_hs, v_rs, v_hs, k_pages, v_pages, slots, T, kvh, num_pages, shift};
    if (row_dtype == 0 && page_dtype == 0) append_launch<float, float>(a, stream);
    else if (row_dtype == 0) append_launch<float, bf16_t>(a, stream);
    else if (page_dtype == 0) append_launch<bf16_t, float>(a, stream);
    else append_launch<bf16_t, bf16_t>(a, stream);
    SPN_LAUNCH_CHECK();
    return SPN_OK;
}
