// khq_paged.hip -- what a server's step does around its attention: the block
// tables and slots of the new tokens, and their rows' front (head norms,
// rotation, cache writes).
#include "khq_paged_internal.h"

namespace khq {
namespace paged {
namespace {

// ------------------------------------------------------------------- plan
// Request s holds has = ceil(kv / P) pages and wants ceil((kv + q) / P); its
// new pages are the free ring's entries from (sum of need before it) on, need =
// want - has, so everything follows from prefix sums over the requests.  Every
// block makes them (4,096 requests are 4 a thread) and then serves its own
// tokens, each finding its request by bisection; block 0 writes what is a
// request's.  Bound: the latency of three dependent loads (lengths, free ring
// or table, store) and of the sums; the bytes are 8 a token.
constexpr int PLAN_THR = 1024;

// Inclusive sums over the block of N values a thread; total: of all threads.
template <int N>
__device__ __forceinline__ void block_scan(long long (&v)[N], long long (&total)[N]) {
    __shared__ long long s_w[N][PLAN_THR / 64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < N; i++) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const long long x = __shfl_up(v[i], o, 64);
            if (lane >= o) v[i] += x;
        }
        if (lane == 63) s_w[i][wv] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        long long before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < PLAN_THR / 64; w++) {
            const long long x = s_w[i][w];
            if (w < wv) before += x;
            all += x;
        }
        v[i] += before;
        total[i] = all;
    }
    __syncthreads();
}

// First index in [0, n) whose s[i + 1] > x (s increasing, s[n] > x).
__device__ __forceinline__ int find(const int* s, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s[mid + 1] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

constexpr int PLAN_SEQS = KHQ_PAGED_MAX_SEQ / PLAN_THR;  // a thread's requests at most

// What the requests of a thread come to.
struct Sums {
    int q[PLAN_SEQS], kv[PLAN_SEQS], has[PLAN_SEQS];
    bool ok[PLAN_SEQS];
    long long end[PLAN_SEQS], upto[PLAN_SEQS], back[PLAN_SEQS];  // inclusive sums
    long long taken, n_back, refused;                           // of all requests
    int head, count;
};

__device__ __forceinline__ void plan_sums(const PlanArgs& a, int per, Sums& s) {
    s.count = min(max(a.state[1], 0), a.n_pages);
    s.head = a.state[0] % a.n_pages;
    if (s.head < 0) s.head += a.n_pages;
    long long v[1] = {0}, t[1];
#pragma unroll
    for (int i = 0; i < PLAN_SEQS; i++) {
        const int sq = threadIdx.x * per + i;
        s.q[i] = i < per && sq < a.n_seq ? a.q_len[sq] : 0;
        s.kv[i] = i < per && sq < a.n_seq ? max(a.kv_len[sq], 0) : 0;
        s.has[i] = (int)(((long long)s.kv[i] + a.page_size - 1) / a.page_size);
        v[0] += max(s.q[i], 0);
        s.end[i] = v[0];
    }
    const long long own = v[0];
    block_scan<1>(v, t);
    long long w[2] = {0, 0}, tw[2];
    int need[PLAN_SEQS];
#pragma unroll
    for (int i = 0; i < PLAN_SEQS; i++) {
        s.end[i] += v[0] - own;
        const long long want = ((long long)s.kv[i] + max(s.q[i], 0) + a.page_size - 1) / a.page_size;
        s.ok[i] = s.q[i] > 0 && want <= a.table_ld && s.end[i] <= a.n_tok;
        need[i] = s.ok[i] ? (int)(want - s.has[i]) : 0;
        w[0] += need[i];
        w[1] += s.q[i] < 0 ? min(s.has[i], a.table_ld) : 0;
        s.upto[i] = w[0];
        s.back[i] = w[1];
    }
    const long long own0 = w[0], own1 = w[1];
    block_scan<2>(w, tw);
    long long x[2] = {0, 0}, tx[2];
#pragma unroll
    for (int i = 0; i < PLAN_SEQS; i++) {
        s.upto[i] += w[0] - own0;
        s.back[i] += w[1] - own1;
        if (need[i] > 0 && s.upto[i] > s.count) s.ok[i] = false;
        x[0] += s.ok[i] ? need[i] : 0;
        x[1] += s.q[i] > 0 && !s.ok[i] ? 1 : 0;
        s.upto[i] -= need[i];  // exclusive
        s.back[i] -= s.q[i] < 0 ? min(s.has[i], a.table_ld) : 0;
    }
    block_scan<2>(x, tx);
    s.taken = tx[0];
    s.refused = tx[1];
    s.n_back = tw[1];
}

// What kv_len and state become.
__device__ __forceinline__ void plan_commit(const PlanArgs& a, int per, const Sums& s) {
#pragma unroll
    for (int i = 0; i < PLAN_SEQS; i++) {
        const int sq = threadIdx.x * per + i;
        if (i >= per || sq >= a.n_seq) continue;
        a.kv_out[sq] = s.ok[i] ? s.kv[i] + s.q[i] : (s.q[i] < 0 ? 0 : s.kv[i]);
    }
    if (threadIdx.x == 0) {
        a.state_out[0] = (int)((s.head + s.taken) % a.n_pages);
        a.state_out[1] = (int)min((long long)a.n_pages, s.count - s.taken + s.n_back);
    }
}

// commit: kv_out and state_out are written here (they are not the inputs, or
// there is one block).
__global__ __launch_bounds__(PLAN_THR) void plan_kernel(PlanArgs a, int per, int tok_per_block,
                                                        int commit) {
    extern __shared__ int s_mem[];
    int* s_cu = s_mem;                    // first rows, [n_seq + 1]
    int* s_pre = s_cu + a.n_seq + 1;      // new pages before a request's, -1: no slots
    int* s_back = s_pre + a.n_seq;        // pages given back before a request's, [n_seq + 1]
    Sums s;
    plan_sums(a, per, s);
    const int tid = threadIdx.x;
    if (tid == 0) {
        s_cu[0] = 0;
        s_back[a.n_seq] = (int)min(s.n_back, (long long)INT32_MAX);
    }
#pragma unroll
    for (int i = 0; i < PLAN_SEQS; i++) {
        const int sq = tid * per + i;
        if (i >= per || sq >= a.n_seq) continue;
        const int end = (int)min(s.end[i], (long long)a.n_tok);
        s_cu[sq + 1] = end;
        s_pre[sq] = s.ok[i] ? (int)s.upto[i] : -1;
        s_back[sq] = (int)min(s.back[i], (long long)INT32_MAX);
        if (blockIdx.x == 0) {
            a.cu_q[sq + 1] = end;
            a.seq_kv[sq] = s.ok[i] ? s.kv[i] + s.q[i] : (s.q[i] == 0 ? s.kv[i] : 0);
        }
    }
    if (blockIdx.x == 0 && tid == 0) {
        a.cu_q[0] = 0;
        a.status[0] = (int)s.refused;
    }
    __syncthreads();
    const int n_rows = s_cu[a.n_seq];
    const int t_end = min(a.n_tok, (int)(blockIdx.x + 1) * tok_per_block);
    for (int t = blockIdx.x * tok_per_block + tid; t < t_end; t += PLAN_THR) {
        int pos = 0, slot = -1;
        if (t < n_rows) {
            const int sq = find(s_cu, a.n_seq, t);
            const int kv = max(a.kv_len[sq], 0);
            pos = (int)((long long)kv + (t - s_cu[sq]));
            const int pre = s_pre[sq];
            if (pre >= 0) {
                const int has = (int)(((long long)kv + a.page_size - 1) / a.page_size);
                const int pg = pos / a.page_size, in = pos - pg * a.page_size;
                int* entry = a.table + (size_t)sq * a.table_ld + pg;
                int page;
                if (pg < has) {
                    page = *entry;
                } else {
                    page = a.free_pages[(int)(((long long)s.head + pre + (pg - has)) % a.n_pages)];
                    if (in == 0) *entry = page;  // a new page's first token is a new token
                }
                if ((unsigned)page < (unsigned)a.n_pages) slot = page * a.page_size + in;
            }
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
    if (blockIdx.x == 0) {
        // ended requests' pages behind the free ones (entries that no new page is read from)
        const int room = a.n_pages - s.count, n_back = min(s_back[a.n_seq], room);
        for (int j = tid; j < n_back; j += PLAN_THR) {
            const int sq = find(s_back, a.n_seq, j);
            a.free_pages[(int)(((long long)s.head + s.count + j) % a.n_pages)] =
                a.table[(size_t)sq * a.table_ld + (j - s_back[sq])];
        }
    }
    if (commit) {
        __syncthreads();  // kv_len read by every token
        if (blockIdx.x == 0) plan_commit(a, per, s);
    }
}

__global__ __launch_bounds__(PLAN_THR) void plan_commit_kernel(PlanArgs a, int per) {
    Sums s;
    plan_sums(a, per, s);
    plan_commit(a, per, s);
}

// ------------------------------------------------------------------- rows
template <typename T>
struct Vec8 {
    typedef T type __attribute__((ext_vector_type(8), aligned(2)));
};

// One wavefront a token head at a time.
template <typename T, int D>
__global__ __launch_bounds__(64) void rows_kernel(RowsArgs a) {
    __shared__ float s_x[D];
    const khq_rows& r = a.r;
    const int row = blockIdx.x, lane = threadIdx.x;
    const int nq = r.q ? r.H_q : 0, nk = r.k ? r.H_kv : 0;
    const int hd = blockIdx.y;
    const int pos = r.positions ? r.positions[row] : r.pos0 + row;
    long long slot = -1;
    if (a.p.k) {
        slot = r.slots[row];
        if (slot >= (long long)a.p.n_pages * a.p.page_size) slot = -1;
    }
    const long long at = slot < 0 ? 0
                                  : slot / a.p.page_size * a.p.page_stride +
                                        slot % a.p.page_size * a.p.token_stride;
    if (hd >= nq + nk) {  // values
        if (slot < 0) return;
        const int h = hd - nq - nk;
        const T* src = (const T*)r.v + row * r.v_token + h * r.v_head;
        T* dst = (T*)a.p.v + at + h * a.p.head_stride;
        for (int i = lane; i < D; i += 64) dst[i] = src[i];
        return;
    }
    const bool is_q = hd < nq;
    const int h = is_q ? hd : hd - nq;
    const T* src = is_q ? (const T*)r.q + row * r.q_token + h * r.q_head
                        : (const T*)r.k + row * r.k_token + h * r.k_head;
    const float* w = is_q ? r.q_weight : r.k_weight;
    float ss = 0.f;
    for (int i = lane; i < D; i += 64) {
        const float x = (float)src[i];
        ss += x * x;
    }
    for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o, 64);
    const float inv = 1.0f / sqrtf(ss / (float)D + r.eps);
    for (int i = lane; i < D; i += 64) {
        float x = (float)src[i] * inv;
        if (w) x *= w[i];
        if (!is_q && r.k_normed)
            ((T*)r.k_normed)[row * r.k_normed_token + h * r.k_normed_head + i] = (T)x;
        s_x[i] = r.round_norm ? (float)(T)x : x;
    }
    __syncthreads();
    const int half = r.rotary_dim / 2;
    for (int i = lane; i < D; i += 64) {
        float y = s_x[i];
        if (i < r.rotary_dim) {
            const int m = i < half ? i : i - half;
            double rev = (double)pos * a.freq[m];
            rev -= rint(rev);
            const float c = __builtin_amdgcn_cosf((float)rev), sn = __builtin_amdgcn_sinf((float)rev);
            const float o = s_x[i < half ? i + half : i - half];
            y = i < half ? y * c - o * sn : y * c + o * sn;
        }
        const T t = (T)y;
        if (is_q) ((T*)r.q_out)[row * r.q_out_token + h * r.q_out_head + i] = t;
        else {
            if (r.k_out) ((T*)r.k_out)[row * r.k_out_token + h * r.k_out_head + i] = t;
            if (slot >= 0) ((T*)a.p.k)[at + h * a.p.head_stride + i] = t;
        }
    }
}

}  // namespace

hipError_t launch_plan(const PlanArgs& a, bool in_place, hipStream_t st) {
    const int per = (a.n_seq + PLAN_THR - 1) / PLAN_THR;
    // one block while its tokens are few
    const int tok = 4 * PLAN_THR;
    const int blocks = a.n_tok > tok ? (a.n_tok + tok - 1) / tok : 1;
    const bool later = in_place && blocks > 1;
    const size_t lds = (3 * (size_t)a.n_seq + 2) * sizeof(int);
    hipLaunchKernelGGL(plan_kernel, dim3(blocks), dim3(PLAN_THR), lds, st, a, per, tok, later ? 0 : 1);
    if (later) hipLaunchKernelGGL(plan_commit_kernel, dim3(1), dim3(PLAN_THR), 0, st, a, per);
    return hipGetLastError();
}

template <typename T>
static hipError_t rows_of(const RowsArgs& a, hipStream_t st) {
    const khq_rows& r = a.r;
    const int heads = (r.q ? r.H_q : 0) + (r.k ? r.H_kv : 0) + (a.p.k ? r.H_kv : 0);
    const dim3 grid(r.n, heads);
    switch (r.head_dim) {
        case 64: hipLaunchKernelGGL((rows_kernel<T, 64>), grid, dim3(64), 0, st, a); break;
        case 128: hipLaunchKernelGGL((rows_kernel<T, 128>), grid, dim3(64), 0, st, a); break;
        default: hipLaunchKernelGGL((rows_kernel<T, 256>), grid, dim3(64), 0, st, a); break;
    }
    return hipGetLastError();
}

hipError_t launch_rows(const RowsArgs& a, hipStream_t st) {
    return a.r.dtype == KHQ_FP16 ? rows_of<fp16>(a, st) : rows_of<bf16>(a, st);
}

}  // namespace paged
}  // namespace khq
