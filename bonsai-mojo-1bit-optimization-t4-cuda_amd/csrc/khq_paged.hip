// khq_paged.hip -- what a server's step does around its attention: the block
// tables and slots of the new tokens, and their rows' front (head norms,
// rotation, cache writes).
#include "khq_mfma_util.h"
#include "khq_paged_internal.h"

#include <algorithm>

namespace khq {
namespace paged {
namespace {

// ------------------------------------------------------------------- plan
// Request s holds has = ceil(kv / P) pages and wants ceil((kv + q) / P); its
// new pages are the free ring's entries from (sum of need before it) on, need =
// want - has, so everything follows from prefix sums over the requests.  Every
// block makes them and then serves its own tokens, each finding its request by
// bisection; block 0 writes what is a request's.  Bound: latency, of the launch,
// of three dependent loads (lengths, free ring or table) and of two sums; the
// bytes are 8 a token.  So the sums are of 32 bits, saturating just past the
// largest one that matters, and the divisions multiplications.  64 decoding
// requests: 3.6 us; 512 requests with 50,000 new tokens: 7.0.
constexpr int PLAN_THR = 1024;
constexpr int PLAN_SEQS = KHQ_PAGED_MAX_SEQ / PLAN_THR;  // a thread's requests at most
// Tokens of a block where there are several; up to PLAN_ONE one block takes
// them all if the step is in place (several blocks then need a second launch,
// as none may change the lengths while another reads them).
constexpr int PLAN_TOK = 1024;
constexpr int PLAN_ONE = 8192;

// a + b of values up to most <= 2^31, at most most.
__device__ __forceinline__ uint32_t sat(uint32_t a, uint32_t b, uint32_t most) { return min(a + b, most); }

// Saturating inclusive sums over the lanes: within rows of 16, then rows to the
// right of lanes 15, 31 and 47.  (Each step is a register operation; shuffles
// through LDS and a walk over the wavefronts' sums made three such sums of 512
// requests 3 us of a plan's 8.)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_from(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t scan_row(uint32_t v, uint32_t most) {
    v = sat(v, dpp_from<0x111, 0xF>(v), most);  // row_shr 1, 2, 4, 8
    v = sat(v, dpp_from<0x112, 0xF>(v), most);
    v = sat(v, dpp_from<0x114, 0xF>(v), most);
    return sat(v, dpp_from<0x118, 0xF>(v), most);
}
__device__ __forceinline__ uint32_t scan(uint32_t v, uint32_t most) {
    v = scan_row(v, most);
    v = sat(v, dpp_from<0x142, 0xA>(v), most);  // row_bcast 15, 31
    return sat(v, dpp_from<0x143, 0xC>(v), most);
}
// Saturating sums of v[i] over the threads before this one; s_w: a word a wavefront.
constexpr int PLAN_WAVES = PLAN_THR / 64;
static_assert(PLAN_WAVES <= 16, "their sums are a row of lanes");
template <int N>
__device__ __forceinline__ void sum_before(uint32_t (&v)[N], uint32_t most, uint32_t (*s_w)[PLAN_WAVES]) {
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[i] = scan(v[i], most);
        if (lane == 63) s_w[i][wv] = v[i];
        v[i] = dpp_from<0x138, 0xF>(v[i]);  // the lane before's
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t w = scan_row(lane < wv ? s_w[i][lane] : 0u, most);  // (wv is below 16)
        v[i] = sat(v[i], (uint32_t)__builtin_amdgcn_readlane((int)w, 15), most);
    }
}

// First index in [0, n) whose s[i + 1] > x, s increasing (the last if none; s[n] is not read).
__device__ __forceinline__ int find(const int* s, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s[mid + 1] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
__device__ __forceinline__ int pages_of(const PlanArgs& a, int tokens) {  // any tokens >= 0
    return a.by_page.div((uint32_t)tokens + (uint32_t)(a.page_size - 1));
}
// Entry i of the free ring, i counted from its first (i <= n_pages).
__device__ __forceinline__ int ring(const PlanArgs& a, int head, int i) {
    const uint32_t x = (uint32_t)head + (uint32_t)i;
    return (int)(x >= (uint32_t)a.n_pages ? x - (uint32_t)a.n_pages : x);
}

// What requests thread * per + i come to.
struct Sums {
    int q[PLAN_SEQS], kv[PLAN_SEQS], has[PLAN_SEQS];
    bool ok[PLAN_SEQS];
    uint32_t end[PLAN_SEQS], pre[PLAN_SEQS], back[PLAN_SEQS];  // rows up to it; pages before it
    int head, count;
};
struct PlanLds {
    uint32_t w[3][PLAN_WAVES];
    int taken, refused, n_back;  // of all requests, after the next barrier
};

__device__ __forceinline__ void plan_sums(const PlanArgs& a, int per, Sums& s, PlanLds& lds) {
    const uint32_t most_q = (uint32_t)a.n_tok + 1, most_p = (uint32_t)a.n_pages + 1;
    const int head = a.state[0], count = a.state[1];
    if (threadIdx.x == 0) lds.taken = lds.refused = lds.n_back = 0;
    uint32_t of_rows[1] = {0};
    uint32_t& rows = of_rows[0];
#pragma unroll
    for (int i = 0; i < PLAN_SEQS; i++) {
        const int sq = threadIdx.x * per + i;
        const bool in = i < per && sq < a.n_seq;
        s.q[i] = in ? a.q_len[sq] : 0;
        s.kv[i] = in ? max(a.kv_len[sq], 0) : 0;
        s.has[i] = pages_of(a, s.kv[i]);
        rows = sat(rows, min((uint32_t)max(s.q[i], 0), most_q), most_q);
    }
    s.head = head % a.n_pages;
    s.head += s.head < 0 ? a.n_pages : 0;
    s.count = min(max(count, 0), a.n_pages);
    sum_before(of_rows, most_q, lds.w);
    uint32_t need = 0, back = 0, mine[PLAN_SEQS];
#pragma unroll
    for (int i = 0; i < PLAN_SEQS; i++) {
        rows = sat(rows, min((uint32_t)max(s.q[i], 0), most_q), most_q);
        s.end[i] = rows;
        // (table_ld * page_size is below 2^31)
        s.ok[i] = s.q[i] > 0 && s.kv[i] <= a.table_ld * a.page_size - s.q[i] && rows <= (uint32_t)a.n_tok;
        mine[i] = s.ok[i] ? pages_of(a, s.kv[i] + s.q[i]) - s.has[i] : 0;
        s.pre[i] = need;
        s.back[i] = back;
        need = sat(need, min(mine[i], most_p), most_p);
        back = sat(back, s.q[i] < 0 ? min((uint32_t)min(s.has[i], a.table_ld), most_p) : 0, most_p);
    }
    uint32_t before[2] = {need, back};
    sum_before(before, most_p, lds.w + 1);
    const uint32_t need0 = before[0], back0 = before[1];
    int taken = 0, refused = 0;
#pragma unroll
    for (int i = 0; i < PLAN_SEQS; i++) {
        s.pre[i] = sat(s.pre[i], need0, most_p);
        s.back[i] = sat(s.back[i], back0, most_p);
        const uint32_t upto = sat(s.pre[i], min(mine[i], most_p), most_p);
        if (mine[i] > 0 && upto > (uint32_t)s.count) s.ok[i] = false;
        if (mine[i] > 0 && s.ok[i]) taken = (int)upto;
        refused += s.q[i] > 0 && !s.ok[i] ? 1 : 0;
    }
    if (taken) atomicMax(&lds.taken, taken);
    if (refused) atomicAdd(&lds.refused, refused);
    if (threadIdx.x == blockDim.x - 1) lds.n_back = (int)sat(back, back0, most_p);
}

// What kv_len and state become.
__device__ __forceinline__ void plan_commit(const PlanArgs& a, int per, const Sums& s, const PlanLds& lds) {
#pragma unroll
    for (int i = 0; i < PLAN_SEQS; i++) {
        const int sq = threadIdx.x * per + i;
        if (i >= per || sq >= a.n_seq) continue;
        a.kv_out[sq] = s.ok[i] ? s.kv[i] + s.q[i] : (s.q[i] < 0 ? 0 : s.kv[i]);
    }
    if (threadIdx.x == 0) {
        a.state_out[0] = ring(a, s.head, lds.taken) % a.n_pages;
        const int left = s.count - lds.taken;
        a.state_out[1] = left + min(a.n_pages - left, lds.n_back);
    }
}

// commit: kv_out and state_out are written here (they are not the inputs, or
// there is one block).
__global__ __launch_bounds__(PLAN_THR) void plan_kernel(PlanArgs a, int per, int tok_per_block,
                                                        int commit) {
    extern __shared__ int s_mem[];
    __shared__ PlanLds lds;
    int* s_cu = s_mem;                // first rows, [n_seq + 1]
    int* s_back = s_cu + a.n_seq + 1;  // pages given back before a request's
    int* s_pre = s_back + a.n_seq;     // new pages before a request's, -1: no slots
    int* s_kv = s_pre + a.n_seq;
    Sums s;
    plan_sums(a, per, s, lds);
    const int tid = threadIdx.x, thr = blockDim.x;
    if (tid == 0) s_cu[0] = 0;
#pragma unroll
    for (int i = 0; i < PLAN_SEQS; i++) {
        const int sq = tid * per + i;
        if (i >= per || sq >= a.n_seq) continue;
        const int end = min((int)s.end[i], a.n_tok);
        s_cu[sq + 1] = end;
        s_back[sq] = (int)s.back[i];
        s_pre[sq] = s.ok[i] ? (int)s.pre[i] : -1;
        s_kv[sq] = s.kv[i];
        if (blockIdx.x == 0) {
            a.cu_q[sq + 1] = end;
            a.seq_kv[sq] = s.ok[i] ? s.kv[i] + s.q[i] : (s.q[i] == 0 ? s.kv[i] : 0);
        }
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        a.cu_q[0] = 0;
        a.status[0] = lds.refused;
    }
    // ended requests' pages behind the free ones (entries that no new page is read from)
    const int n_back = min(lds.n_back, a.n_pages - s.count);
    for (int j = blockIdx.x * thr + tid; j < n_back; j += gridDim.x * thr) {
        const int sq = find(s_back, a.n_seq, j);
        a.free_pages[ring(a, s.head, s.count + j)] = a.table[(size_t)sq * a.table_ld + (j - s_back[sq])];
    }
    const int n_rows = s_cu[a.n_seq];
    const int t_end = min(a.n_tok, (int)(blockIdx.x + 1) * tok_per_block);
    for (int t = blockIdx.x * tok_per_block + tid; t < t_end; t += thr) {
        int pos = 0, slot = -1;
        if (t < n_rows) {
            const int sq = find(s_cu, a.n_seq, t), kv = s_kv[sq], pre = s_pre[sq];
            pos = (int)((uint32_t)kv + (uint32_t)(t - s_cu[sq]));
            if (pre >= 0) {
                const int has = pages_of(a, kv), pg = a.by_page.div(pos), in = pos - pg * a.page_size;
                int* entry = a.table + (size_t)sq * a.table_ld + pg;
                int page;
                if (pg < has) {
                    page = *entry;
                } else {
                    page = a.free_pages[ring(a, s.head, pre + (pg - has))];
                    if (in == 0) *entry = page;  // a new page's first token is a new token
                }
                if ((unsigned)page < (unsigned)a.n_pages) slot = page * a.page_size + in;
            }
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
    if (commit && blockIdx.x == 0) plan_commit(a, per, s, lds);
}

__global__ __launch_bounds__(PLAN_THR) void plan_commit_kernel(PlanArgs a, int per) {
    __shared__ PlanLds lds;
    Sums s;
    plan_sums(a, per, s, lds);
    __syncthreads();
    plan_commit(a, per, s, lds);
}

// ------------------------------------------------------------------- rows
// Bound: memory, every value read and written once.  A lane holds 8 dims (16
// bytes) of a head, so a wavefront takes 512 / D heads of one token at a time,
// U times over with all loads in flight before the first sum; a token's heads
// are its queries', its keys' and, with pages, its values', in this order.  The
// angles belong to the token: their sines and cosines are taken once a
// wavefront, while its loads are under way, from revolutions reduced in 64
// bits (a position of 2^18 leaves 32 bits 2 digits of the angle).  8,192 tokens,
// 24 / 4 heads of 256 in fp16: 268 MB in 56 us (4.8 TB/s; a copy runs at 4.9);
// 1,999 of 32 / 8 heads of 128 in bf16, every dim turned: 49 MB in 14.5; 32: 4.
template <typename T>
struct Pack8 {
    typedef T x8 __attribute__((ext_vector_type(8)));
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    typedef uint32_t u4e __attribute__((ext_vector_type(4), aligned(2)));  // a caller's rows
};
constexpr int ROWS_WAVES = 4;

template <typename T, int D, int U>
__global__ __launch_bounds__(64 * ROWS_WAVES) void rows_kernel(RowsArgs a) {
    typedef typename Pack8<T>::x8 x8;
    typedef typename Pack8<T>::u4 u4;
    typedef typename Pack8<T>::u4e u4e;
    constexpr int CH = D / 8, G = 64 / CH;
    const khq_rows& r = a.r;
    const int row = blockIdx.x, lane = threadIdx.x & 63, c = lane % CH;
    const int nq = r.q ? r.H_q : 0, nk = r.k ? r.H_kv : 0, heads = nq + nk + (a.p.k ? nk : 0);
    const int hd0 = ((blockIdx.y * ROWS_WAVES + (threadIdx.x >> 6)) * U) * G + lane / CH;
    u4 x[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int hd = min(hd0 + i * G, heads - 1);
        const T* src = hd < nq ? (const T*)r.q + row * r.q_token + hd * r.q_head
                       : hd < nq + nk
                           ? (const T*)r.k + row * r.k_token + (hd - nq) * r.k_head
                           : (const T*)r.v + row * r.v_token + (hd - nq - nk) * r.v_head;
        x[i] = *reinterpret_cast<const u4e*>(src + 8 * c);
    }
    long long at = -1;  // of the token in the cache
    if (a.p.k) {
        const int slot = r.slots[row], pg = a.by_page.div(max(slot, 0));
        if (slot >= 0 && pg < a.p.n_pages)
            at = pg * a.p.page_stride + (slot - pg * a.p.page_size) * a.p.token_stride;
    }
    const int half = r.rotary_dim >> 1, hc = half >> 3;  // pieces of half the rotated dims
    const bool turns = c < 2 * hc;
    float cs[8], sn[8];
    if (turns) {
        const double pos = (double)(r.positions ? r.positions[row] : r.pos0 + row);
        const int m0 = 8 * (c < hc ? c : c - hc);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            double rev = pos * a.freq[m0 + e];
            rev -= rint(rev);
            cs[e] = __builtin_amdgcn_cosf((float)rev);
            sn[e] = __builtin_amdgcn_sinf((float)rev);
            sn[e] = c < hc ? -sn[e] : sn[e];
        }
    }
    const int other = turns ? (c < hc ? lane + hc : lane - hc) : lane;
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int hd = hd0 + i * G;
        const bool is_q = hd < nq, is_k = !is_q && hd < nq + nk;
        const int h = is_q ? hd : is_k ? hd - nq : hd - nq - nk;
        const x8 xv = __builtin_bit_cast(x8, x[i]);
        float y[8], ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            y[e] = (float)xv[e];
            ss = fmaf(y[e], y[e], ss);
        }
        ss += mu::xor_lane<1>(ss);
        ss += mu::xor_lane<2>(ss);
        ss += mu::xor_lane<4>(ss);
        if constexpr (CH > 8) ss += mu::xor_lane<8>(ss);
        if constexpr (CH > 16) ss += mu::xor_lane<16>(ss);
        const float inv = 1.0f / sqrtf(ss / (float)D + r.eps);
        const float* w = is_q ? r.q_weight : is_k ? r.k_weight : nullptr;
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] *= inv;
        if (w) {
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] *= w[8 * c + e];
        }
        x8 normed;
#pragma unroll
        for (int e = 0; e < 8; e++) normed[e] = (T)y[e];
        if (r.round_norm) {
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = (float)normed[e];
        }
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] = __shfl(y[e], other, 64);
        x8 out;
#pragma unroll
        for (int e = 0; e < 8; e++) out[e] = (T)(turns ? fmaf(z[e], sn[e], y[e] * cs[e]) : y[e]);
        const u4e o = __builtin_bit_cast(u4, out);
        if (is_q) {
            *reinterpret_cast<u4e*>((T*)r.q_out + row * r.q_out_token + h * r.q_out_head + 8 * c) = o;
        } else if (is_k) {
            if (r.k_normed)
                *reinterpret_cast<u4e*>((T*)r.k_normed + row * r.k_normed_token + h * r.k_normed_head + 8 * c) =
                    __builtin_bit_cast(u4, normed);
            if (r.k_out)
                *reinterpret_cast<u4e*>((T*)r.k_out + row * r.k_out_token + h * r.k_out_head + 8 * c) = o;
            if (at >= 0)
                *reinterpret_cast<u4*>((T*)a.p.k + at + h * a.p.head_stride + 8 * c) =
                    __builtin_bit_cast(u4, out);
        } else if (hd < heads && at >= 0) {
            *reinterpret_cast<u4*>((T*)a.p.v + at + h * a.p.head_stride + 8 * c) = x[i];
        }
    }
}

}  // namespace

hipError_t launch_plan(const PlanArgs& a, bool in_place, hipStream_t st) {
    const int per = (a.n_seq + PLAN_THR - 1) / PLAN_THR;
    const int tok = in_place && a.n_tok <= PLAN_ONE ? std::max(a.n_tok, 1) : PLAN_TOK;
    const int blocks = std::max(1, (a.n_tok + tok - 1) / tok);
    // a thread a request or a token
    const int want = std::max(a.n_seq, std::min(a.n_tok, tok));
    const int thr = std::min(PLAN_THR, (want + 63) / 64 * 64);
    const bool later = in_place && blocks > 1;
    const size_t lds = (4 * (size_t)a.n_seq + 1) * sizeof(int);
    const hipError_t e = lds > 32768 ? ensure_dynamic_lds(reinterpret_cast<const void*>(plan_kernel), 66000)
                                     : hipSuccess;
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(plan_kernel, dim3(blocks), dim3(thr), lds, st, a, per, tok, later ? 0 : 1);
    if (later) hipLaunchKernelGGL(plan_commit_kernel, dim3(1), dim3(thr), 0, st, a, per);
    return hipGetLastError();
}

template <typename T, int D>
static hipError_t rows_of(const RowsArgs& a, hipStream_t st) {
    const khq_rows& r = a.r;
    const int heads = (r.q ? r.H_q : 0) + (r.k ? r.H_kv : 0) + (a.p.k ? r.H_kv : 0);
    const int groups = (heads + 512 / D - 1) / (512 / D);
    if (r.n >= 256) {
        hipLaunchKernelGGL((rows_kernel<T, D, 4>), dim3(r.n, (groups + 15) / 16), dim3(256), 0, st, a);
    } else {  // few tokens: a wavefront a group
        hipLaunchKernelGGL((rows_kernel<T, D, 1>), dim3(r.n, (groups + 3) / 4), dim3(256), 0, st, a);
    }
    return hipGetLastError();
}

hipError_t launch_rows(const RowsArgs& a, hipStream_t st) {
    const bool f16 = a.r.dtype == KHQ_FP16;
    switch (a.r.head_dim) {
        case 64: return f16 ? rows_of<fp16, 64>(a, st) : rows_of<bf16, 64>(a, st);
        case 128: return f16 ? rows_of<fp16, 128>(a, st) : rows_of<bf16, 128>(a, st);
        default: return f16 ? rows_of<fp16, 256>(a, st) : rows_of<bf16, 256>(a, st);
    }
}

}  // namespace paged
}  // namespace khq
