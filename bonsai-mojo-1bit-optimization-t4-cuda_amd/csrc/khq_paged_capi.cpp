// khq_paged_capi.cpp -- extern "C" boundary of libkhq_paged.so (declared in
// include/khq_paged.h): every shape, stride and pointer is checked here, before
// anything is launched; what lies on the device (lengths, tables, slots) the
// kernels check.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>
#include <mutex>

#include "khq_paged.h"
#include "khq_paged_internal.h"

namespace {

int rc_of(hipError_t e) { return e == hipSuccess ? 0 : static_cast<int>(e); }

bool dim_ok(int d) { return d == 64 || d == 128 || d == 256; }
bool dtype_ok(int t) { return t == KHQ_FP16 || t == KHQ_BF16; }

bool pages_ok(const khq_pages* p) {
    if (!p || !p->k || !p->v || p->n_pages <= 0 || p->page_size <= 0 || p->H_kv <= 0 ||
        !dim_ok(p->head_dim) || !dtype_ok(p->dtype))
        return false;
    if ((long long)p->n_pages * p->page_size > 0x7fffffffLL) return false;
    if (p->page_stride < 0 || p->token_stride < 0 || p->head_stride < 0) return false;
    // pieces of 16 bytes
    const long long off = (long long)(reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v));
    return (off & 15) == 0 && ((p->page_stride | p->token_stride | p->head_stride) & 7) == 0;
}

}  // namespace

extern "C" {

int khq_paged_plan(const int* q_len, const int* kv_len, int* table, int table_ld,
                   int* free_pages, const int* state, int n_seq, int n_pages, int page_size,
                   int n_tok, int* cu_q, int* seq_kv, int* kv_out, int* state_out, int* status,
                   int* positions, int* slots, hipStream_t stream) {
    if (!q_len || !kv_len || !table || !free_pages || !state || !cu_q || !seq_kv || !kv_out ||
        !state_out || !status || n_seq <= 0 || n_seq > KHQ_PAGED_MAX_SEQ || table_ld <= 0 ||
        n_pages <= 0 || page_size <= 0 || n_tok < 0 || (n_tok > 0 && (!positions || !slots)))
        return -100;
    if (n_pages >= 1 << 30 || n_tok >= 1 << 30) return -100;  // sums of two stay in 32 bits
    if ((long long)n_pages * page_size > 0x7fffffffLL || (long long)table_ld * page_size > 0x7fffffffLL)
        return -100;
    khq::paged::PlanArgs a{q_len, kv_len, table, free_pages, state, cu_q, seq_kv, kv_out, state_out,
                           status, positions, slots, n_seq, table_ld, n_pages, page_size, n_tok,
                           khq::FastDiv(page_size)};
    return rc_of(khq::paged::launch_plan(a, kv_out == kv_len || state_out == state, stream));
}

int khq_qk_norm_rope(const khq_rows* rows, const khq_pages* pages, hipStream_t stream) {
    if (!rows) return -100;
    const khq_rows& r = *rows;
    if (r.n < 0 || !dim_ok(r.head_dim) || !dtype_ok(r.dtype) || !(r.eps >= 0.0f) || (!r.q && !r.k) ||
        (r.q && (!r.q_out || r.H_q <= 0)) || (r.k && r.H_kv <= 0) || r.pos0 < 0)
        return -100;
    if (r.rotary_dim < 0 || r.rotary_dim > r.head_dim || r.rotary_dim % 16 != 0 ||
        (r.rotary_dim > 0 && !(r.theta > 0.0 && std::isfinite(r.theta))))
        return -100;
    if (pages && (!pages_ok(pages) || !r.k || !r.v || !r.slots || pages->H_kv != r.H_kv ||
                  pages->head_dim != r.head_dim || pages->dtype != r.dtype))
        return -100;
    if (pages && ((pages->n_pages > 1 && pages->page_stride < r.head_dim) ||
                  (pages->page_size > 1 && pages->token_stride < r.head_dim) ||
                  (pages->H_kv > 1 && pages->head_stride < r.head_dim)))
        return -100;  // slots that share memory, as an expanded tensor's do
    if (!pages && r.k && !r.k_out && !r.k_normed) return -100;  // nothing to leave the keys in
    if (!r.positions && r.pos0 > 0x7fffffff - r.n) return -100;  // the last position
    if (r.n == 0) return 0;
    khq::paged::RowsArgs a{};
    a.r = r;
    if (pages) {
        a.p = *pages;
        a.by_page = khq::FastDiv(pages->page_size);
    }
    // revolutions a position of each pair, in 64 bits: a table of the last base and width
    static thread_local double freq[128], base = 0;
    static thread_local int width = 0;
    if (r.rotary_dim > 0 && (base != r.theta || width != r.rotary_dim)) {
        for (int i = 0; i < r.rotary_dim / 2; i++)
            freq[i] = std::exp(-2.0 * i / r.rotary_dim * std::log(r.theta)) * 0.15915494309189533577;
        base = r.theta;
        width = r.rotary_dim;
    }
    std::memcpy(a.freq, freq, sizeof(double) * (r.rotary_dim / 2));
    return rc_of(khq::paged::launch_rows(a, stream));
}

static bool attn_sizes_ok(int n_tok, int n_seq, int H_q, int H_kv, int head_dim, int max_q) {
    return n_tok >= 0 && n_seq > 0 && n_seq <= KHQ_PAGED_MAX_SEQ && H_q > 0 && H_kv > 0 &&
           H_q % H_kv == 0 && dim_ok(head_dim) && max_q > 0 && (long long)n_tok * H_q < 1LL << 27 &&
           (long long)n_seq * H_kv <= 1LL << 21;  // a launch's blocks
}

long long khq_paged_attn_ws_bytes(int n_tok, int n_seq, int H_q, int H_kv, int head_dim, int max_q) {
    if (!attn_sizes_ok(n_tok, n_seq, H_q, H_kv, head_dim, max_q)) return -100;
    return (long long)khq::paged::attn_ws_bytes(n_tok, n_seq, H_q, H_kv, head_dim, max_q);
}

int khq_paged_attn(const khq_attn_rows* rows, const khq_pages* pages, hipStream_t stream) {
    if (!rows || !pages_ok(pages)) return -100;
    const khq_attn_rows& r = *rows;
    if (!attn_sizes_ok(r.n_tok, r.n_seq, r.H_q, pages->H_kv, pages->head_dim, r.max_q) || !r.q ||
        !r.out || !r.cu_q || !r.seq_kv || !r.table || r.table_ld <= 0 ||
        (long long)r.table_ld * pages->page_size > 0x7fffffffLL || !std::isfinite(r.scale))
        return -100;
    if (r.n_tok == 0) return 0;
    khq::paged::AttnArgs a{};
    a.r = r;
    a.p = *pages;
    a.n_rep = r.H_q / pages->H_kv;
    a.by_page = khq::FastDiv(pages->page_size);
    a.by_rep = khq::FastDiv(a.n_rep);
    a.by_kv = khq::FastDiv(pages->H_kv);
    const size_t need = khq::paged::attn_ws_bytes(r.n_tok, r.n_seq, r.H_q, pages->H_kv,
                                                  pages->head_dim, r.max_q);
    if (r.ws) {
        if (r.ws_bytes < need || (reinterpret_cast<uintptr_t>(r.ws) & 15)) return -101;
        return rc_of(khq::paged::launch_attn(a, stream));
    }
    // One caller at a time takes the shared workspace and launches: the next one's
    // stream waits for these launches, and its growing it does not come between.
    static std::mutex launching;
    std::lock_guard<std::mutex> lock(launching);
    float* ws = nullptr;
    const hipError_t e = khq::shared_workspace(need, stream, &ws);
    if (e != hipSuccess) return rc_of(e);
    a.r.ws = ws;
    return rc_of(khq::paged::launch_attn(a, stream));
}

}  // extern "C"
