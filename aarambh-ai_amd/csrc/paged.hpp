// Argument blocks and launchers of the paged-cache operators and the logits processor.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.hpp"
#include "paged_rule.hpp"

namespace aarh {

enum ActFmt { ACT_F32 = 0, ACT_F16 = 1, ACT_BF16 = 2 };
enum { KV_BF16 = 3 };  // beside KvFmt: pages only

struct PagePool {
    int fmt, n_kv, hd, page_shift, n_pages;
    void *k, *v;
    uint16_t *ks, *vs;
};

struct PageBatch {
    int nseq, rows, max_rows, max_kv;
    const int32_t *row_off, *kv_len, *tables;
    long long table_ld;
    int32_t* status;
};

struct RopeAppendArgs {
    PagePool pool;
    PageBatch bt;
    int act, n_heads;
    const void *q, *k, *v;
    long long q_ld, k_ld, v_ld;
    void* q_out;
    long long q_out_ld;
    const double* inv_freq;
    int rot, interleaved;
    float attn;
};
int launch_rope_append(const RopeAppendArgs& a, hipStream_t stream);

struct PagedAttnArgs {
    PagePool pool;
    PageBatch bt;
    int act, n_heads, grouped;
    const void* q;
    long long q_ld;
    void* out;
    long long out_ld;
    float scale, softcap;
    int window;
    const float* slopes;
    const int32_t* prefix;
    void* workspace;
};
int launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream);
long long paged_attention_workspace(const PagedAttnArgs& a);

struct LogitsArgs {
    int nseq, R, V;
    const float* x;
    long long ld;
    float* out;
    long long out_ld;
    const uint32_t* hist;
    long long hist_ld;
    const int32_t *hist_len, *prompt_len;
    const float* pen;
    const uint32_t* draft;
    long long draft_ld;
    const int32_t* bias_off;
    const uint32_t* bias_ids;
    const float* bias_vals;
    int n_bias;
    const uint32_t* masks;
    long long mask_ld;
    int n_masks;
    const int32_t* mask_of_row;
};
int launch_process_logits(const LogitsArgs& a, hipStream_t stream);

}  // namespace aarh
