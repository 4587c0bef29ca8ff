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
// so the served ones take a contiguous piece off the top of the stack.
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
        s_len[tid] = len; s_given[tid] = served ? fresh : 0; s_top[tid] = nf - 1 - (int)(end - max(need, 0));
        if (r < a.R) a.lens_out[r] = served ? len + fresh : len;
        if (served && need > 0) atomicMax(&s_taken, (int)end);
        if (tid == PLAN_T - 1) red[0] = incl;
        __syncthreads();
        carry += red[0];
        for (long e = tid; e < (long)n * a.width; e += PLAN_T) {
            const int q = (int)(e / a.width), i = (int)(e - (long)q * a.width);
            plan_emit(a, r0 + q, i, s_len[q], s_given[q], s_top[q]);
        }
        __syncthreads();
    }
    if (tid == 0) *a.num_free_out = nf - s_taken;
}

struct ReleaseArgs { const uint8_t* done; int* lens; int* table; long ld; int* stack; int* num_free; int R, W, num_pages, shift; };

// One workgroup, a wave per request.  The pages go back so that page 0 of the first ended request lies on top of the stack: a plan for the
// same requests and lengths takes the same pages again.  Two passes: how many pages, then where.
__global__ __launch_bounds__(PLAN_T) void release_kernel(ReleaseArgs a) {
    __shared__ int red[16], cnt[PLAN_T], s_total;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int nf = min(max(*a.num_free, 0), a.num_pages);
    int total = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int carry = 0;
        for (int r0 = 0; r0 < a.R; r0 += PLAN_T) {
            const int n = min(PLAN_T, a.R - r0);
            cnt[tid] = 0;
            __syncthreads();
            for (int q = w; q < n; q += 16) {
                const int r = r0 + q;
                if (!a.done[r]) continue;
                const int held = (int)min(pages_of(a.lens[r], a.shift), (long)a.W);
                int c = 0;
                for (int j = 0; j < held; j += 64) c += __popcll(__ballot(j + lane < held && page_ok(a.table[r * a.ld + j + lane], a.num_pages)));
                if (lane == 0) cnt[q] = c;
            }
            __syncthreads();
            const int mine = cnt[tid], incl = block_scan(mine, red);
            if (tid == PLAN_T - 1) s_total = incl;
            cnt[tid] = carry + incl - mine;
            __syncthreads();
            carry += s_total;
            if (pass == 1) {
                for (int q = w; q < n; q += 16) {
                    const int r = r0 + q;
                    if (!a.done[r]) continue;
                    const int held = (int)min(pages_of(a.lens[r], a.shift), (long)a.W);
                    int at = nf + total - 1 - cnt[q];
                    for (int j = 0; j < held; j += 64) {
                        const int id = j + lane < held ? a.table[r * a.ld + j + lane] : -1;
                        const bool ok = page_ok(id, a.num_pages);
                        const unsigned long long m = __ballot(ok);
                        const int to = at - __popcll(m & ((1ull << lane) - 1));
                        if (ok && page_ok(to, a.num_pages)) a.stack[to] = id;      // more pages than the pool has: a page was held twice
                        if (j + lane < held) a.table[r * a.ld + j + lane] = -1;
                        at -= __popcll(m);
                    }
                    if (lane == 0) a.lens[r] = 0;
                }
            }
            __syncthreads();
        }
        if (pass == 0) total = carry;
    }
    if (tid == 0) *a.num_free = min(nf + total, a.num_pages);
}

struct AppendArgs {
    const void* k; const void* v; long k_rs, k_hs, v_rs, v_hs; void* k_pages; void* v_pages; const long long* slots; long T; int kvh, num_pages, shift;
};

template <typename T> __device__ __forceinline__ float load1(const T* p) {
    if constexpr (sizeof(T) == 2) return bf2f(*p); else return *p;
}

// A thread moves one element of a key row and of the value row of the same note.
template <typename S, typename D>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
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

int log2_page(int page) {   // -1: not a power of two in [8, 4096]
    for (int s = 3; s <= 12; ++s) if (page == 1 << s) return s;
    return -1;
}

}  // namespace

extern "C" int spn_paged_plan(const int* lens, const int* fresh, int* block_table, long bt_ld, const int* free_pages, const int* num_free,
                              int* lens_out, int* num_free_out, long long* slots, int R, int W, int num_pages, int page, int width,
                              hipStream_t stream) {
    const int shift = log2_page(page);
    SPN_REQUIRE(lens && fresh && block_table && free_pages && num_free && lens_out && num_free_out && slots, "spn_paged_plan: null buffer");
    SPN_REQUIRE(shift >= 0, "spn_paged_plan: the page size must be a power of two in [8, 4096]");
    SPN_REQUIRE(R > 0 && W > 0 && num_pages > 0 && width > 0 && bt_ld >= W, "spn_paged_plan: bad sizes");
    SPN_REQUIRE((long)R * W < (1L << 31) && ((long)W << shift) < (1L << 31) && (long)R * width < (1L << 31), "spn_paged_plan: sizes pass 2^31");
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(PLAN_T), 0, stream,
                       PlanArgs{lens, fresh, block_table, bt_ld, free_pages, num_free, lens_out, num_free_out, slots, R, W, num_pages, shift, width});
    SPN_LAUNCH_CHECK();
    return SPN_OK;
}

extern "C" int spn_paged_release(const uint8_t* done, int* lens, int* block_table, long bt_ld, int* free_pages, int* num_free, int R, int W,
                                 int num_pages, int page, hipStream_t stream) {
    const int shift = log2_page(page);
    SPN_REQUIRE(done && lens && block_table && free_pages && num_free, "spn_paged_release: null buffer");
    SPN_REQUIRE(shift >= 0, "spn_paged_release: the page size must be a power of two in [8, 4096]");
    SPN_REQUIRE(R > 0 && W > 0 && num_pages > 0 && bt_ld >= W && (long)R * W < (1L << 31), "spn_paged_release: bad sizes");
    hipLaunchKernelGGL(release_kernel, dim3(1), dim3(PLAN_T), 0, stream, ReleaseArgs{done, lens, block_table, bt_ld, free_pages, num_free, R, W, num_pages, shift});
    SPN_LAUNCH_CHECK();
    return SPN_OK;
}

extern "C" int spn_paged_append(const void* k, const void* v, int row_dtype, long k_rs, long k_hs, long v_rs, long v_hs, void* k_pages, void* v_pages,
                                int page_dtype, const long long* slots, long T, int kvh, int num_pages, int page, hipStream_t stream) {
    const int shift = log2_page(page);
    SPN_REQUIRE(k && v && k_pages && v_pages && slots, "spn_paged_append: null buffer");
    SPN_REQUIRE((row_dtype | page_dtype) >> 1 == 0, "spn_paged_append: dtype codes are 0 (fp32) and 1 (bf16)");
    SPN_REQUIRE(shift >= 0, "spn_paged_append: the page size must be a power of two in [8, 4096]");
    SPN_REQUIRE(T > 0 && kvh > 0 && num_pages > 0 && T * kvh < (1L << 31), "spn_paged_append: bad sizes");
    const AppendArgs a{k, v, k_rs, k_hs, v_rs, v_hs, k_pages, v_pages, slots, T, kvh, num_pages, shift};
    const dim3 grid(cdiv(T * kvh * HEAD, 256)), block(256);
    if (row_dtype == 0 && page_dtype == 0) hipLaunchKernelGGL((append_kernel<float, float>), grid, block, 0, stream, a);
    else if (row_dtype == 0) hipLaunchKernelGGL((append_kernel<float, bf16_t>), grid, block, 0, stream, a);
    else if (page_dtype == 0) hipLaunchKernelGGL((append_kernel<bf16_t, float>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((append_kernel<bf16_t, bf16_t>), grid, block, 0, stream, a);
    SPN_LAUNCH_CHECK();
    return SPN_OK;
}
