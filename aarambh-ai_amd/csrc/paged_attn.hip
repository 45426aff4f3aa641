// Attention of a call's new rows over the paged key / value cache.
//
// One wave per (row, query head): 64 keys at a time, one a lane, with the running maximum and sum
// of the softmax; then each lane adds its output dimensions over the 64 keys.
#include "device_common.hpp"
#include "paged.hpp"

namespace aarh {

namespace {

template <typename T, typename C, bool I8, int HD>
__global__ __launch_bounds__(64) void paged_attn_kernel(PagedAttnArgs a) {
    const int lane = threadIdx.x, i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    __shared__ float s_q[HD], s_p[64];
    PageSeq s;
    if (!page_seq(a.bt.row_off, a.bt.kv_len, b, a.bt.rows, a.bt.max_rows, a.bt.max_kv, &s)) {
        if (a.bt.status && lane == 0) atomicOr(&a.bt.status[b], PAGE_SEQ_BAD_LENGTH);
        return;
    }
    if (i >= s.rows) return;
    const int p = s.kv_len - s.rows + i;
    const int kvh = a.grouped ? h / (a.n_heads / a.pool.n_kv) : h % a.pool.n_kv;
    const int pre = a.prefix ? min(a.prefix[b], s.kv_len) : 0;
    const T* q = (const T*)a.q + (long long)(s.row0 + i) * a.q_ld + h * HD;
    for (int d = lane; d < HD; d += 64) s_q[d] = (float)q[d];
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    const int low = a.window ? max(0, p - a.window + 1) : 0;
    const int end = max(p + 1, pre);
    float m = -INFINITY, l = 0.f, o[HD / 64] = {};
    bool bad = false;
    const int32_t* table = a.bt.tables + b * a.bt.table_ld;
    for (int t0 = 0; t0 < end; t0 += 64) {
        if (t0 >= pre && t0 + 64 <= low) continue;
        const int t = t0 + lane;
        const bool vis = t < end && ((t <= p && t >= low) || t < pre);
        int page = -1;
        if (vis) {
            page = page_of(table, t, a.pool.page_shift, a.pool.n_pages);
            bad |= page < 0;
        }
        const int in_page = t & ((1 << a.pool.page_shift) - 1);
        const size_t head = (size_t)max(page, 0) * a.pool.n_kv + kvh;
        const size_t base = (head << a.pool.page_shift) * HD + (size_t)(in_page >> 5) * (PAGE_BLK * HD);
        const size_t tok = (head << a.pool.page_shift) + in_page;
        float x = -INFINITY, vsc = 0.f;
        __syncthreads();
        if (page >= 0) {
            x = 0.f;
            for (int d = 0; d < HD; d++) x += s_q[d] * (float)((const C*)a.pool.k)[base + page_k_at(t & 31, d, HD, I8)];
            if (I8) {
                x *= (float)__builtin_bit_cast(_Float16, a.pool.ks[tok]);
                vsc = (float)__builtin_bit_cast(_Float16, a.pool.vs[tok]);
            }
            x *= a.scale;
            if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
            x += slope * (float)(t - p);
        }
        const float mx = fmaxf(m, wave_max_f32(x));
        const float use = mx == -INFINITY ? 0.f : mx;
        const float e = __expf(x - use), alpha = __expf(m - use);
        l = l * alpha + wave_sum_f32(e);
        m = mx;
        s_p[lane] = I8 ? e * vsc : e;
        __syncthreads();
        for (int k = 0; k < HD / 64; k++) o[k] *= alpha;
        for (int j = 0; j < 64; j++) {
            const unsigned at_lo = __builtin_amdgcn_readlane((int)(uint32_t)base, j);
            const unsigned at_hi = __builtin_amdgcn_readlane((int)(uint32_t)(base >> 32), j);
            const size_t at = ((size_t)at_hi << 32) | at_lo;
            const int pg = __builtin_amdgcn_readlane(page, j);
            if (pg < 0) continue;
            for (int k = 0; k < HD / 64; k++)
                o[k] += s_p[j] * (float)((const C*)a.pool.v)[at + page_v_at((t0 + j) & 31, lane + 64 * k, HD, I8)];
        }
    }
    T* out = (T*)a.out + (long long)(s.row0 + i) * a.out_ld + h * HD;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    for (int k = 0; k < HD / 64; k++) out[lane + 64 * k] = (T)(o[k] * inv);
    if (bad && a.bt.status) atomicOr(&a.bt.status[b], PAGE_SEQ_BAD_PAGE);
}

template <typename T, typename C, bool I8>
int launch_hd(const PagedAttnArgs& a, hipStream_t stream) {
    const dim3 grid(a.bt.max_rows, a.n_heads, a.bt.nseq);
    if (a.pool.hd == 128)
        hipLaunchKernelGGL((paged_attn_kernel<T, C, I8, 128>), grid, dim3(64), 0, stream, a);
    else
        hipLaunchKernelGGL((paged_attn_kernel<T, C, I8, 64>), grid, dim3(64), 0, stream, a);
    return note_error(hipGetLastError());
}

}  // namespace

long long paged_attention_workspace(const PagedAttnArgs&) { return 0; }

int launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
    if (a.act == ACT_F32)
        return a.pool.fmt == KV_INT8 ? launch_hd<float, int8_t, true>(a, stream)
                                     : launch_hd<float, _Float16, false>(a, stream);
    if (a.act == ACT_F16)
        return a.pool.fmt == KV_INT8 ? launch_hd<_Float16, int8_t, true>(a, stream)
                                     : launch_hd<_Float16, _Float16, false>(a, stream);
    return launch_hd<__bf16, __bf16, false>(a, stream);
}

}  // namespace aarh
