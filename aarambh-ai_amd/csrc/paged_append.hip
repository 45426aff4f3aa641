// Rotary positions of a call's new rows and their append to the pages of the key / value cache.
//
// (x, y) -> attn * (x cos - y sin, y cos + x sin) for the pairs of the first `rot` dimensions of every head,
// angle = position * inv_freq.  A stream of positions far into a context needs the angle in f64:
// its f32 rounding alone is 2^-24 * angle.  So the turns (angle / 2 pi) are formed in f64, reduced
// to [-1/2, 1/2], and only the remainder goes through f32 sine and cosine.
//
// One workgroup takes one 32-token block of one sequence's new positions: the block is what a
// page stores contiguously (V transposed within it), and its angles serve every head.  The
// workgroup's head slots are either kv heads (key and value rows through LDS, whole 16-byte pieces
// out) or query heads (straight from load to store).
#include <cfloat>

#include "device_common.hpp"
#include "paged.hpp"

namespace aarh {

namespace {

constexpr int RA_THREADS = 256;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f(__bf16 v) { return (float)v; }

// 8 consecutive elements
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int per = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += per) {
        const vec v = *(const vec*)(p + i);
#pragma unroll
        for (int j = 0; j < per; j++) x[i + j] = to_f(v[j]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int per = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += per) {
        vec v;
#pragma unroll
        for (int j = 0; j < per; j++) v[j] = (T)x[i + j];
        *(vec*)(p + i) = v;
    }
}

// Rotates one unit of a head and stores it.  Half layout: unit u < rot / 16 is the pair of pieces 8 u and
// rot / 2 + 8 u, later units are pieces past rot.  Interleaved: unit u is piece 8 u.
template <typename T, typename Put>
__device__ __forceinline__ void rotate_unit(const T* src, int u, int rot, bool inter, const float2_t* cs, Put put) {
    float x[8];
    if (inter) {
        load8(src + 8 * u, x);
        if (8 * u < rot) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2_t c = cs[4 * u + i / 2];
                const float a = x[i], b = x[i + 1];
                x[i] = a * c[0] - b * c[1];
                x[i + 1] = b * c[0] + a * c[1];
            }
        }
        put(8 * u, x);
        return;
    }
    const int pairs = rot >> 4;
    if (u >= pairs) {
        const int d = rot + 8 * (u - pairs);
        load8(src + d, x);
        put(d, x);
        return;
    }
    float y[8], r[8];
    load8(src + 8 * u, x);
    load8(src + (rot >> 1) + 8 * u, y);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float2_t c = cs[8 * u + i];
        r[i] = x[i] * c[0] - y[i] * c[1];
        y[i] = y[i] * c[0] + x[i] * c[1];
    }
    put(8 * u, r);
    put((rot >> 1) + 8 * u, y);
}

template <typename T, int KVF, int HD>
__global__ __launch_bounds__(RA_THREADS) void rope_append_kernel(RopeAppendArgs a, int kv_per, int q_per) {
    typedef typename std::conditional<KVF == KV_F16, _Float16, __bf16>::type C;  // 16-bit pools
    constexpr int LDK = HD + 4;  // f32 row of LDS
    __shared__ float2_t s_cs[PAGE_BLK * (HD / 2)];
    __shared__ float s_k[PAGE_BLK * LDK], s_v[PAGE_BLK * LDK];
    __shared__ float s_sc[2][PAGE_BLK];
    const int tid = threadIdx.x, b = blockIdx.z;
    PageSeq s;
    if (!page_seq(a.bt.row_off, a.bt.kv_len, b, a.bt.rows, a.bt.max_rows, a.bt.max_kv, &s)) {
        if (a.bt.status && blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) atomicOr(&a.bt.status[b], PAGE_SEQ_BAD_LENGTH);
        return;
    }
    const int pos0 = s.kv_len - s.rows;
    const int blk = (pos0 >> 5) + blockIdx.x;
    const int p0 = max(blk * PAGE_BLK, pos0), p1 = min((blk + 1) * PAGE_BLK, s.kv_len);
    if (p0 >= p1) return;
    const int n = p1 - p0;  // new tokens of this block; the first is row r0
    const long long r0 = s.row0 + (p0 - pos0);
    const int half = a.rot >> 1;
    const bool inter = a.interleaved != 0;
    for (int i = tid; i < n * half; i += RA_THREADS) {
        const int t = i / half, j = i - t * half;
        const double turns = (double)(p0 + t) * (a.inv_freq[j] * 0.15915494309189533577);
        float sn, cn;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cn);
        s_cs[t * half + j] = float2_t{cn * a.attn, sn * a.attn};
    }
    __syncthreads();
    const int units = inter ? HD / 8 : (a.rot >> 4) + ((HD - a.rot) >> 3);
    const int kv_slots = (a.pool.n_kv + kv_per - 1) / kv_per;
    if ((int)blockIdx.y >= kv_slots) {
        const int h0 = (blockIdx.y - kv_slots) * q_per, h1 = min(h0 + q_per, a.n_heads);
        for (int i = tid; i < n * (h1 - h0) * units; i += RA_THREADS) {
            const int u = i % units, th = i / units, h = h0 + th % (h1 - h0), t = th / (h1 - h0);
            T* dst = (T*)a.q_out + (r0 + t) * a.q_out_ld + h * HD;
            rotate_unit((const T*)a.q + (r0 + t) * a.q_ld + h * HD, u, a.rot, inter, s_cs + t * half,
                        [&](int d, const float(&x)[8]) { store8(dst + d, x); });
        }
        return;
    }
    const int page = page_of(a.bt.tables + b * a.bt.table_ld, p0, a.pool.page_shift, a.pool.n_pages);
    if (page < 0) {
        if (a.bt.status && tid == 0) atomicOr(&a.bt.status[b], PAGE_SEQ_BAD_PAGE);
        return;
    }
    const int t0 = p0 & (PAGE_BLK - 1);
    const int blk_in_page = (p0 & ((1 << a.pool.page_shift) - 1)) >> 5;
    for (int h = blockIdx.y * kv_per; h < min((int)(blockIdx.y + 1) * kv_per, a.pool.n_kv); h++) {
        const size_t head = (size_t)page * a.pool.n_kv + h;
        const size_t base = (head << a.pool.page_shift) * HD + (size_t)blk_in_page * (PAGE_BLK * HD);
        for (int i = tid; i < n * units; i += RA_THREADS) {
            const int u = i % units, t = i / units;
            rotate_unit((const T*)a.k + (r0 + t) * a.k_ld + h * HD, u, a.rot, inter, s_cs + t * half,
                        [&](int d, const float(&x)[8]) { store8(s_k + t * LDK + d, x); });
        }
        for (int i = tid; i < n * (HD / 8); i += RA_THREADS) {
            const int d = i % (HD / 8) * 8, t = i / (HD / 8);
            float x[8];
            load8((const T*)a.v + (r0 + t) * a.v_ld + h * HD + d, x);
            store8(s_v + t * LDK + d, x);
        }
        __syncthreads();
        if constexpr (KVF == KV_INT8) {
            // absmax scale of a (token, kv head): code = x / scale from the f32 scale, kept as fp16
            for (int row = tid >> 6; row < 2 * n; row += RA_THREADS / 64) {
                const float* src = (row & 1 ? s_v : s_k) + (row >> 1) * LDK;
                float m = fabsf(src[tid & 63]);
                if (HD == 128) m = fmaxf(m, fabsf(src[64 + (tid & 63)]));
                m = wave_max_f32(m);
                const float sc = m <= FLT_EPSILON ? 1.0f : m / 127.0f;
                if ((tid & 63) == 0) {
                    s_sc[row & 1][row >> 1] = sc;
                    (row & 1 ? a.pool.vs : a.pool.ks)[(head << a.pool.page_shift) + blk_in_page * PAGE_BLK + t0 + (row >> 1)] =
                        __builtin_bit_cast(uint16_t, (_Float16)sc);
                }
            }
            __syncthreads();
            auto code = [](float x, float sc) { return (int8_t)fminf(fmaxf(roundf(x / sc), -127.0f), 127.0f); };
            for (int i = tid; i < n * (HD / 8); i += RA_THREADS) {
                const int d = i % (HD / 8) * 8, t = i / (HD / 8);
                uint64_t w = 0;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    w |= (uint64_t)(uint8_t)code(s_k[t * LDK + d + j], s_sc[0][t]) << (8 * j);
                *(uint64_t*)((int8_t*)a.pool.k + base + page_k_at(t0 + t, d, HD, true)) = w;
            }
            for (int i = tid; i < n * HD; i += RA_THREADS) {
                const int t = i / HD, d = i % HD;
                ((int8_t*)a.pool.v)[base + page_v_at(t0 + t, d, HD, true)] = code(s_v[t * LDK + d], s_sc[1][t]);
            }
        } else {
            for (int i = tid; i < n * (HD / 8); i += RA_THREADS) {
                const int d = i % (HD / 8) * 8, t = i / (HD / 8);
                float x[8];
                load8(s_k + t * LDK + d, x);
                store8((C*)a.pool.k + base + page_k_at(t0 + t, d, HD, false), x);
            }
            for (int i = tid; i < n * HD; i += RA_THREADS) {
                const int t = i / HD, d = i % HD;
                ((C*)a.pool.v)[base + page_v_at(t0 + t, d, HD, false)] = (C)s_v[t * LDK + d];
            }
        }
        __syncthreads();
    }
}

template <typename T, int KVF>
int launch_rope_hd(const RopeAppendArgs& a, int blocks, int kv_per, int q_per, hipStream_t stream) {
    const dim3 grid(blocks, (a.pool.n_kv + kv_per - 1) / kv_per + (a.n_heads + q_per - 1) / q_per, a.bt.nseq);
    if (a.pool.hd == 128)
        hipLaunchKernelGGL((rope_append_kernel<T, KVF, 128>), grid, dim3(RA_THREADS), 0, stream, a, kv_per, q_per);
    else
        hipLaunchKernelGGL((rope_append_kernel<T, KVF, 64>), grid, dim3(RA_THREADS), 0, stream, a, kv_per, q_per);
    return note_error(hipGetLastError());
}

}  // namespace

int launch_rope_append(const RopeAppendArgs& a, hipStream_t stream) {
    const int blocks = (a.bt.max_rows + 30) / PAGE_BLK + 1;  // blocks that max_rows positions can touch
    const int kv_per = 1, q_per = 8;
    if (a.act == ACT_F32)
        return a.pool.fmt == KV_INT8 ? launch_rope_hd<float, KV_INT8>(a, blocks, kv_per, q_per, stream)
                                     : launch_rope_hd<float, KV_F16>(a, blocks, kv_per, q_per, stream);
    if (a.act == ACT_F16)
        return a.pool.fmt == KV_INT8 ? launch_rope_hd<_Float16, KV_INT8>(a, blocks, kv_per, q_per, stream)
                                     : launch_rope_hd<_Float16, KV_F16>(a, blocks, kv_per, q_per, stream);
    return launch_rope_hd<__bf16, KV_BF16>(a, blocks, kv_per, q_per, stream);
}

}  // namespace aarh
