// Penalties for repeated tokens, biases and grammar masks on logits rows.
//
// A workgroup takes a piece of the vocabulary for all rows of one sequence.  It counts the
// piece's tokens in the sequence's history into LDS (integer atomics: any order, one result),
// then streams the rows: row t has the counts of the history and of the first t proposals,
// which are added between the rows.
#include "device_common.hpp"
#include "paged.hpp"

namespace aarh {

namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_MAX = 8192;               // vocabulary piece of a workgroup
constexpr uint32_t LG_PROMPT = 0x80000000u;  // the token stands in the prompt; the rest counts the others

__global__ __launch_bounds__(LG_THREADS) void process_logits_kernel(LogitsArgs a, int piece) {
    extern __shared__ uint32_t lds[];
    uint32_t* s_cnt = lds;
    uint32_t* s_bias = lds + piece;  // index + 1 of the last bias entry of a token, relative to the sequence's first
    const int tid = threadIdx.x, b = blockIdx.y;
    const int v0 = blockIdx.x * piece, n = min(piece, a.V - v0);
    const bool biased = a.bias_off != nullptr;
    for (int i = tid; i < piece; i += LG_THREADS) {
        s_cnt[i] = 0;
        if (biased) s_bias[i] = 0;
    }
    __syncthreads();
    if (a.hist) {
        const int len = (int)min((long long)max(a.hist_len[b], 0), a.hist_ld);
        const int prompt = a.prompt_len ? a.prompt_len[b] : 0;
        const uint32_t* h = a.hist + b * a.hist_ld;
        for (int i = tid; i < len; i += LG_THREADS) {
            const uint32_t id = h[i] - (uint32_t)v0;
            if (id >= (uint32_t)n) continue;
            if (i < prompt) atomicOr(&s_cnt[id], LG_PROMPT);
            else atomicAdd(&s_cnt[id], 1u);
        }
    }
    int b0 = 0;
    if (biased) {
        b0 = max(a.bias_off[b], 0);
        const int b1 = min(a.bias_off[b + 1], a.n_bias);
        for (int i = b0 + tid; i < b1; i += LG_THREADS) {
            const uint32_t id = a.bias_ids[i] - (uint32_t)v0;
            if (id < (uint32_t)n) atomicMax(&s_bias[id], (uint32_t)(i - b0 + 1));
        }
    }
    __syncthreads();
    const float rep = a.pen ? a.pen[3 * b] : 1.f, pres = a.pen ? a.pen[3 * b + 1] : 0.f, freq = a.pen ? a.pen[3 * b + 2] : 0.f;
    for (int t = 0; t < a.R; t++) {
        const long long row = (long long)b * a.R + t;
        const float* x = a.x + row * a.ld + v0;
        float* y = a.out + row * a.out_ld + v0;
        const int mi = a.masks ? a.mask_of_row[row] : -1;
        const bool none = mi < -1 || mi >= a.n_masks;
        const uint32_t* mk = mi >= 0 && !none ? a.masks + mi * a.mask_ld : nullptr;
        for (int i = tid; i < n; i += LG_THREADS) {
            float v = x[i];
            const uint32_t c = s_cnt[i];
            if (c) {
                v = v > 0.f ? v / rep : v * rep;
                const uint32_t k = c & ~LG_PROMPT;
                if (k) v = v - pres - freq * (float)k;
            }
            if (biased && s_bias[i]) v += a.bias_vals[b0 + s_bias[i] - 1];
            if (none || (mk && !((mk[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1u))) v = -INFINITY;
            y[i] = v;
        }
        if (t + 1 < a.R && a.draft) {
            const uint32_t id = a.draft[b * a.draft_ld + t] - (uint32_t)v0;
            if (id < (uint32_t)n) {
                __syncthreads();
                if (tid == 0) s_cnt[id] += 1u;
                __syncthreads();
            }
        }
    }
}

}  // namespace

int launch_process_logits(const LogitsArgs& a, hipStream_t stream) {
    const int piece = 1024;
    const dim3 grid((a.V + piece - 1) / piece, a.nseq);
    hipLaunchKernelGGL(process_logits_kernel, grid, dim3(LG_THREADS), (size_t)piece * (a.bias_off ? 8 : 4), stream, a, piece);
    return note_error(hipGetLastError());
}

}  // namespace aarh
