// Penalties for repeated tokens, biases and grammar masks on logits rows.
//
// A workgroup takes a piece of the vocabulary for all rows of one sequence.  It counts the
// piece's tokens in the sequence's history into LDS (integer atomics: any order, one result),
// then streams the rows: row t has the counts of the history and of the first t proposals,
// which are added between the rows.
//
// Bound by the rows' bytes, read and written once, and in small calls by the latency of the history and of
// the rows one after another.  So a piece is one 16-byte run a thread (pieces of 2, 4 or 8 runs measured 10 - 110% slower:
// fewer workgroups, more rows' latencies in a row), the rows are loaded LG_ROWS at a time with their mask
// words, the first ones before the history is counted, and the history four words a load.
// Measured: one row of 32000 3.6 us; 32 x 5 rows of 32000 with histories of 3000, biases and masks 14 us (2.9 TB/s); 64 x 4 rows
// of 128000 with histories of 8000 and 300 biases 52 us (5.0 TB/s, a large copy's rate).
#include "device_common.hpp"
#include "paged.hpp"

namespace aarh {

namespace {

constexpr int LG_THREADS = 512;
constexpr uint32_t LG_PROMPT = 0x80000000u;  // the token stands in the prompt; the rest counts the others

constexpr int LG_PIECE = 4 * LG_THREADS;  // vocabulary entries of a workgroup
constexpr int LG_ROWS = 4;                 // rows loaded at once

// four values at any 4-byte boundary (one load or store: the memory pipeline asks for no more)
typedef float float4u_t __attribute__((ext_vector_type(4), aligned(4)));

template <bool BIAS>
__global__ __launch_bounds__(LG_THREADS) void process_logits_kernel(LogitsArgs a) {
    __shared__ __attribute__((aligned(16))) uint32_t s_cnt[LG_PIECE];
    // index + 1 of the last bias entry of a token, relative to the sequence's first
    __shared__ __attribute__((aligned(16))) uint32_t s_bias[BIAS ? LG_PIECE : 4];
    const int tid = threadIdx.x, b = blockIdx.y;
    const int v0 = blockIdx.x * LG_PIECE, n = min(LG_PIECE, a.V - v0), e = 4 * tid;
    const bool all = e + 4 <= n;
    // this thread's values of rows t0 .. t0 + LG_ROWS - 1 and their mask bits (1: token e + j may follow)
    float4_t v[LG_ROWS];
    uint32_t ok[LG_ROWS];
    auto load = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < LG_ROWS; k++) {
            if (t0 + k >= a.R) break;
            const long long row = (long long)b * a.R + t0 + k;
            const float* x = a.x + row * a.ld + v0 + e;
            if (all) {
                v[k] = __builtin_nontemporal_load((const float4u_t*)x);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) v[k][j] = e + j < n ? x[j] : 0.f;
            }
            ok[k] = 15u;
            if (a.masks) {
                const int mi = a.mask_of_row[row];
                if (mi >= 0 && mi < a.n_masks) {
                    if (e < n) ok[k] = a.masks[mi * a.mask_ld + ((v0 + e) >> 5)] >> ((v0 + e) & 31);
                } else if (mi != -1) {
                    ok[k] = 0;
                }
            }
        }
    };
    load(0);
    *(uint4*)&s_cnt[e] = uint4{0, 0, 0, 0};
    if (BIAS) *(uint4*)&s_bias[e] = uint4{0, 0, 0, 0};
    __syncthreads();
    if (a.hist) {
        const int len = (int)min((long long)max(a.hist_len[b], 0), a.hist_ld);
        const int prompt = a.prompt_len ? a.prompt_len[b] : 0;
        const uint32_t* h = a.hist + b * a.hist_ld;
        auto count = [&](uint32_t word, int i) __attribute__((always_inline)) {
            const uint32_t id = word - (uint32_t)v0;
            if (id >= (uint32_t)n) return;
            if (i < prompt) atomicOr(&s_cnt[id], LG_PROMPT);
            else atomicAdd(&s_cnt[id], 1u);
        };
        // four words to a load from the first 16-byte boundary on
        const int head = min(len, (int)((16 - ((uintptr_t)h & 15)) & 15) / 4), quads = (len - head) / 4;
        if (tid < head) count(h[tid], tid);
        const int tail = head + 4 * quads + tid;
        if (tail < len && tid < 4) count(h[tail], tail);
        const uint4* hq = (const uint4*)(h + head);
        for (int q0 = 0; q0 < quads; q0 += 4 * LG_THREADS) {
            uint4 w[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int q = q0 + k * LG_THREADS + tid;
                if (q < quads) w[k] = hq[q];
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int q = q0 + k * LG_THREADS + tid, i = head + 4 * q;
                if (q >= quads) continue;
                count(w[k].x, i);
                count(w[k].y, i + 1);
                count(w[k].z, i + 2);
                count(w[k].w, i + 3);
            }
        }
    }
    int b0 = 0;
    if (BIAS) {
        b0 = max(a.bias_off[b], 0);
        const int b1 = min(a.bias_off[b + 1], a.n_bias);
        for (int i = b0 + tid; i < b1; i += LG_THREADS) {
            const uint32_t id = a.bias_ids[i] - (uint32_t)v0;
            if (id < (uint32_t)n) atomicMax(&s_bias[id], (uint32_t)(i - b0 + 1));
        }
    }
    const float rep = a.pen ? a.pen[3 * b] : 1.f, pres = a.pen ? a.pen[3 * b + 1] : 0.f, freq = a.pen ? a.pen[3 * b + 2] : 0.f;
    const float inv = 1.f / rep;
    __syncthreads();
    float4_t bias = {0.f, 0.f, 0.f, 0.f};
    if (BIAS) {
        const uint4 k = *(const uint4*)&s_bias[e];
        if (k.x) bias[0] = a.bias_vals[b0 + k.x - 1];
        if (k.y) bias[1] = a.bias_vals[b0 + k.y - 1];
        if (k.z) bias[2] = a.bias_vals[b0 + k.z - 1];
        if (k.w) bias[3] = a.bias_vals[b0 + k.w - 1];
    }
    for (int t0 = 0; t0 < a.R; t0 += LG_ROWS) {
        if (t0) load(t0);
#pragma unroll
        for (int k = 0; k < LG_ROWS; k++) {
            const int t = t0 + k;
            if (t >= a.R) break;
            const uint4 c4 = *(const uint4*)&s_cnt[e];
            const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
            float4_t z = v[k];
            if (c4.x | c4.y | c4.z | c4.w) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    // z / rep, rounded as a division: the quotient by the reciprocal, put right by its remainder
                    float q = z[j] * inv;
                    const float fixed = fmaf(fmaf(-q, rep, z[j]), inv, q);
                    q = fabsf(q) < INFINITY ? fixed : q;
                    const float s = z[j] > 0.f ? q : z[j] * rep;
                    const uint32_t times = c[j] & ~LG_PROMPT;
                    z[j] = c[j] ? s : z[j];
                    z[j] = times ? z[j] - pres - freq * (float)times : z[j];
                }
            }
            if (BIAS) z += bias;
#pragma unroll
            for (int j = 0; j < 4; j++) z[j] = (ok[k] >> j) & 1u ? z[j] : -INFINITY;
            float* y = a.out + ((long long)b * a.R + t) * a.out_ld + v0 + e;
            if (all) {
                __builtin_nontemporal_store((float4u_t)z, (float4u_t*)y);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (e + j < n) y[j] = z[j];
            }
            if (t + 1 < a.R && a.draft) {
                const uint32_t id = a.draft[b * a.draft_ld + t] - (uint32_t)v0;
                if (id < (uint32_t)n) {  // (the same for every thread)
                    __syncthreads();
                    if (tid == 0) s_cnt[id] += 1u;
                    __syncthreads();
                }
            }
        }
    }
}

}  // namespace

int launch_process_logits(const LogitsArgs& a, hipStream_t stream) {
    const dim3 grid((a.V + LG_PIECE - 1) / LG_PIECE, a.nseq);
    if (a.bias_off) hipLaunchKernelGGL((process_logits_kernel<true>), grid, dim3(LG_THREADS), 0, stream, a);
    else hipLaunchKernelGGL((process_logits_kernel<false>), grid, dim3(LG_THREADS), 0, stream, a);
    return note_error(hipGetLastError());
}

}  // namespace aarh
