// Attention of one new row per request over its paged key / value cache (the serving form of spn_attn_fwd: causal, one query).
//   o[r, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(s_j - max s),   s_j = scale q[r, h] . k_j - slope_h (len_r - 1 - j)
// over the rows j < len_r that lie on a page; a request without any has zeros.
#include "common.h"
#include "paged_index.h"

using namespace spn_paged;

namespace {

struct PagedAttnArgs {
    const void* q; long q_rs, q_hs; const void* kp; const void* vp; const int* table; long ld; const int* lens; const float* slopes;
    void* o; long o_rs, o_hs; int R, h, kvh, W, num_pages, shift; float scale;
};

template <typename T> __device__ __forceinline__ float load1(const T* p) {
    if constexpr (sizeof(T) == 2) return bf2f(*p); else return *p;
}

// One wave per (request, head), a lane per dimension, a row at a time.
template <typename T>
__global__ __launch_bounds__(64) void paged_attn_kernel(PagedAttnArgs a) {
    const int r = blockIdx.x, hi = blockIdx.y, lane = threadIdx.x, kh = hi / (a.h / a.kvh);
    const int n = rows_of(a.lens[r], a.W, a.shift);
    const float q = load1((const T*)a.q + r * a.q_rs + hi * a.q_hs + lane) * a.scale;
    const float slope = a.slopes ? a.slopes[hi] : 0.f;
    float m = -__builtin_inff(), l = 0.f, acc = 0.f;
    for (int j = 0; j < n; ++j) {
        const int id = a.table[r * a.ld + (j >> a.shift)];
        if (!page_ok(id, a.num_pages)) continue;
        const long at = row_offset(id, kh, j & ((1 << a.shift) - 1), a.kvh, a.shift) + lane;
        const float s = wave_sum(q * load1((const T*)a.kp + at)) - slope * (float)(n - 1 - j);
        const float mn = fmaxf(m, s), c = m == mn ? 1.f : __expf(m - mn), p = __expf(s - mn);
        l = l * c + p; acc = acc * c + p * load1((const T*)a.vp + at);
        m = mn;
    }
    const float o = l > 0.f ? acc / l : (l == 0.f ? 0.f : l);
    T* to = (T*)a.o + r * a.o_rs + hi * a.o_hs + lane;
    if constexpr (sizeof(T) == 2) *to = f2bf(o); else *to = o;
}

}  // namespace

extern "C" int spn_paged_attn(const void* q, long q_rs, long q_hs, const void* k_pages, const void* v_pages, int dtype, const int* block_table, long bt_ld,
                              const int* lens, const float* slopes, void* o, long o_rs, long o_hs, int R, int h, int kvh, int W, int num_pages,
                              int page, float scale, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    int shift = -1;
    for (int s = 3; s <= 12; ++s) if (page == 1 << s) shift = s;
    SPN_REQUIRE(q && k_pages && v_pages && block_table && lens && o, "spn_paged_attn: null buffer");
    SPN_REQUIRE(dtype == 0 || dtype == 1, "spn_paged_attn: dtype codes are 0 (fp32) and 1 (bf16)");
    SPN_REQUIRE(shift >= 0, "spn_paged_attn: the page size must be a power of two in [8, 4096]");
    SPN_REQUIRE(R > 0 && h > 0 && kvh > 0 && h % kvh == 0 && W > 0 && num_pages > 0 && bt_ld >= W && ((long)W << shift) < (1L << 31), "spn_paged_attn: bad sizes");
    const PagedAttnArgs a{q, q_rs, q_hs, k_pages, v_pages, block_table, bt_ld, lens, slopes, o, o_rs, o_hs, R, h, kvh, W, num_pages, shift, scale};
    if (dtype == 1) hipLaunchKernelGGL(paged_attn_kernel<bf16_t>, dim3(R, h), dim3(64), 0, stream, a);
    else hipLaunchKernelGGL(paged_attn_kernel<float>, dim3(R, h), dim3(64), 0, stream, a);
    SPN_LAUNCH_CHECK();
    return SPN_OK;
}

// scratch of spn_paged_attn
extern "C" size_t spn_paged_attn_workspace_bytes(int R, int h, int kvh, int W, int page) { return 0; }
