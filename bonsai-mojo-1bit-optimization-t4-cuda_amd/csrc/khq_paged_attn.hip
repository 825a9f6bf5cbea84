// khq_paged_attn.hip -- attention of new tokens over a paged cache.
#include "khq_paged_internal.h"

namespace khq {
namespace paged {
namespace {

// One wavefront a (row, head): the keys one after the other, running maximum
// and sum.
template <typename T, int D>
__global__ __launch_bounds__(64) void attn_row_kernel(AttnArgs a) {
    const khq_attn_rows& r = a.r;
    const int row = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x;
    int lo = 0, hi = r.n_seq;  // the last sequence whose first row is not past row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (r.cu_q[mid] <= row) lo = mid;
        else hi = mid;
    }
    const int first = r.cu_q[lo], end = r.cu_q[lo + 1];
    if (row < first || row >= end) return;
    const long long cap = (long long)r.table_ld * a.p.page_size;
    const int kv = (int)min((long long)max(r.seq_kv[lo], 0), cap);
    const int vis = min(kv, kv - (end - first) + (row - first) + 1);
    constexpr int N = D / 64;
    float q[N], acc[N], m = -INFINITY, l = 0.f;
    const int h = hq / a.n_rep;
    for (int i = 0; i < N; i++) {
        q[i] = (float)((const T*)r.q)[row * r.q_token + hq * r.q_head + lane * N + i] * r.scale;
        acc[i] = 0.f;
    }
    for (int k = 0; k < vis; k++) {
        const int page = r.table[(size_t)lo * r.table_ld + k / a.p.page_size];
        if ((unsigned)page >= (unsigned)a.p.n_pages) {
            l = NAN;
            continue;
        }
        const long long at = page * a.p.page_stride + k % a.p.page_size * a.p.token_stride +
                             h * a.p.head_stride + lane * N;
        float s = 0.f;
        for (int i = 0; i < N; i++) s += q[i] * (float)((const T*)a.p.k)[at + i];
        for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
        const float mn = fmaxf(m, s);
        const float f = m == mn ? 1.f : expf(m - mn), p = expf(s - mn);
        m = mn;
        l = l * f + p;
        for (int i = 0; i < N; i++) acc[i] = acc[i] * f + p * (float)((const T*)a.p.v)[at + i];
    }
    for (int i = 0; i < N; i++) {
        float o = vis > 0 ? acc[i] / l : 0.f;
        if (r.gate)
            o /= 1.f + expf(-(float)((const T*)r.gate)[row * r.gate_token + hq * r.gate_head + lane * N + i]);
        ((T*)r.out)[row * r.out_token + hq * r.out_head + lane * N + i] = (T)o;
    }
}

}  // namespace

size_t attn_ws_bytes(int, int, int, int, int, int) { return 0; }

template <typename T>
static hipError_t attn_of(const AttnArgs& a, hipStream_t st) {
    const dim3 grid(a.r.n_tok, a.r.H_q);
    switch (a.p.head_dim) {
        case 64: hipLaunchKernelGGL((attn_row_kernel<T, 64>), grid, dim3(64), 0, st, a); break;
        case 128: hipLaunchKernelGGL((attn_row_kernel<T, 128>), grid, dim3(64), 0, st, a); break;
        default: hipLaunchKernelGGL((attn_row_kernel<T, 256>), grid, dim3(64), 0, st, a); break;
    }
    return hipGetLastError();
}

hipError_t launch_attn(const AttnArgs& a, hipStream_t st) {
    return a.p.dtype == KHQ_FP16 ? attn_of<fp16>(a, st) : attn_of<bf16>(a, st);
}

}  // namespace paged
}  // namespace khq
