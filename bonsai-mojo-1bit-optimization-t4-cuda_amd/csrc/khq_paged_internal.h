// khq_paged_internal.h -- argument blocks and launchers of the paged cache
// (khq_paged.hip, khq_paged_attn.hip) for its C ABI (khq_paged_capi.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "khq_internal.h"
#include "khq_paged.h"

namespace khq {

// The device workspace that libkhq_hip.so's launchers share (one a device,
// grown on demand, ordered between streams, kept for captured graphs).
hipError_t shared_workspace(size_t bytes, hipStream_t stream, float** out);

namespace paged {

typedef _Float16 fp16;
typedef __bf16 bf16;

struct PlanArgs {
    const int* q_len;
    const int* kv_len;
    int* table;
    int* free_pages;
    const int* state;
    int *cu_q, *seq_kv, *kv_out, *state_out, *status, *positions, *slots;
    int n_seq, table_ld, n_pages, page_size, n_tok;
    FastDiv by_page;  // page_size
};
// in_place: kv_out is kv_len or state_out is state.
hipError_t launch_plan(const PlanArgs& a, bool in_place, hipStream_t st);

struct RowsArgs {
    khq_rows r;
    khq_pages p;        // k = NULL: none
    FastDiv by_page;    // page_size
    double freq[128];   // revolutions a position, of each dim pair
};
hipError_t launch_rows(const RowsArgs& a, hipStream_t st);

struct AttnArgs {
    khq_attn_rows r;  // ws set
    khq_pages p;
    int n_rep;
    FastDiv by_page, by_rep, by_kv;  // page_size, n_rep, H_kv
};
hipError_t launch_attn(const AttnArgs& a, hipStream_t st);
size_t attn_ws_bytes(int n_tok, int n_seq, int H_q, int H_kv, int head_dim, int max_q);

}  // namespace paged
}  // namespace khq
