// Rotary positions of a call's new rows and their append to the pages of the key / value cache.
//
// (x, y) -> attn * (x cos - y sin, y cos + x sin) for the pairs of the first `rot` dimensions of every head,
// angle = position * inv_freq.  A stream of positions far into a context needs the angle in f64:
// its f32 rounding alone is 2^-24 * angle.  So the turns (angle / 2 pi) are formed in f64, reduced
// to [-1/2, 1/2], and only the remainder goes through f32 sine and cosine.
//
// One workgroup takes one 32-token block of one sequence's new positions (the block is what a page stores
// together) and either keys, values or queries of a few heads: keys and queries need the block's angles, values
// do not, and separate workgroups keep the wait for one from holding up the other.  Keys and queries go from load
// to store in 16-byte pieces whose loads are under way while the angles are made.  Values change places
// with their tokens: a thread loads eight dimensions of eight tokens and stores eight tokens of eight dimensions.
// INT8 pools take keys and values of a head together through LDS, for the largest value of a row.
// Bound by the bytes in large calls and by one round of dependent loads (lengths, page, rows) in small ones.
// Measured (bf16 in and out, head size 128): 4 prompts of 2048, 32 query heads on 8 kv heads, 48 us (3.4 TB/s);
// 512 rows 8.7 us; one row 4.2 us.  A workgroup for all three with the values turned through LDS takes 82 us.
#include <cfloat>

#include "device_common.hpp"
#include "paged.hpp"

namespace aarh {

namespace {

constexpr int RA_THREADS = 256;

// 8 consecutive elements
typedef float float8_t __attribute__((ext_vector_type(8)));
template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));
template <typename T>
__device__ __forceinline__ vec8<T> load8(const T* p) {
    if constexpr (sizeof(T) == 4) {
        const float4_t a = *(const float4_t*)p, b = *(const float4_t*)(p + 4);
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        return *(const vec8<T>*)p;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, float8_t x) {
    if constexpr (sizeof(T) == 4) {
        *(float4_t*)p = __builtin_shufflevector(x, x, 0, 1, 2, 3);
        *(float4_t*)(p + 4) = __builtin_shufflevector(x, x, 4, 5, 6, 7);
    } else {
        *(vec8<T>*)p = __builtin_convertvector(x, vec8<T>);
    }
}

// The units of a head: half layout, rot / 16 pairs of pieces 8 u and rot / 2 + 8 u and then the pieces past rot;
// interleaved, hd / 8 pieces.
struct Units {
    int pairs, all, rot;
    bool inter;
};
template <typename T>
struct Piece2 {  // as loaded: half the registers of f32 values
    vec8<T> x, y;
};
template <typename T>
__device__ __forceinline__ Piece2<T> unit_load(const T* src, int u, const Units& un) {
    const bool pair = !un.inter && u < un.pairs;
    const int d = un.inter || pair ? 8 * u : un.rot + 8 * (u - un.pairs);
    Piece2<T> p;
    p.x = load8(src + d);
    p.y = pair ? load8(src + d + (un.rot >> 1)) : p.x;
    return p;
}
// Rotates a loaded unit by its token's angles and hands its pieces to put(dimension, values).
template <typename T, typename Put>
__device__ __forceinline__ void unit_turn(const Piece2<T>& raw, int u, const Units& un, const float2_t* cs, Put put) {
    struct {
        float8_t x, y;
    } p = {__builtin_convertvector(raw.x, float8_t), __builtin_convertvector(raw.y, float8_t)};
    if (un.inter) {
        if (8 * u < un.rot) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2_t c = cs[4 * u + i / 2];
                const float a = p.x[i], b = p.x[i + 1];
                p.x[i] = a * c[0] - b * c[1];
                p.x[i + 1] = b * c[0] + a * c[1];
            }
        }
        put(8 * u, p.x);
    } else if (u < un.pairs) {
        float8_t r;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float2_t c = cs[8 * u + i];
            r[i] = p.x[i] * c[0] - p.y[i] * c[1];
            p.y[i] = p.y[i] * c[0] + p.x[i] * c[1];
        }
        put(8 * u, r);
        put((un.rot >> 1) + 8 * u, p.y);
    } else {
        put(un.rot + 8 * (u - un.pairs), p.x);
    }
}

// kv heads of a workgroup (16-bit pools; query workgroups take twice as many) and units of a thread under way.
// Four prompts of 2048 / 512 rows: 2 and 2 48 / 8.7 us, 2 and 4 61 / 8.8, 4 and 2 56 / 11.4, 4 and 4 62 / 11.2.
constexpr int RA_HEADS = 2;
constexpr int RA_AHEAD = 2;

template <typename T, int KVF, int HD>
__global__ __launch_bounds__(RA_THREADS) void rope_append_kernel(RopeAppendArgs a, int kv_slots) {
    constexpr bool I8 = KVF == KV_INT8;
    typedef typename std::conditional<KVF == KV_BF16, __bf16, _Float16>::type C;  // 16-bit pools
    constexpr int LDK = HD + 4;  // f32 row of LDS (INT8)
    __shared__ float2_t s_cs[PAGE_BLK * (HD / 2)];
    __shared__ __attribute__((aligned(16))) float s_k[I8 ? PAGE_BLK * LDK : 4], s_v[I8 ? PAGE_BLK * LDK : 4];
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
    Units un;
    un.rot = a.rot;
    un.inter = a.interleaved != 0;
    un.pairs = a.rot >> 4;
    un.all = un.inter ? HD / 8 : un.pairs + ((HD - a.rot) >> 3);
    // slots: keys (INT8: keys and values), then values, then queries
    const int v_slots = I8 ? 0 : kv_slots;
    const int slot = blockIdx.y;
    const bool keys = slot < kv_slots, values = !keys && slot < kv_slots + v_slots;
    int page = 0;
    if (keys | values) page = page_of(a.bt.tables + b * a.bt.table_ld, p0, a.pool.page_shift, a.pool.n_pages);
    const int t0 = p0 & (PAGE_BLK - 1);
    const int in_page = (p0 & ((1 << a.pool.page_shift) - 1)) >> 5;
    auto block_of = [&](int h) { return (((size_t)page * a.pool.n_kv + h) << a.pool.page_shift) + (size_t)in_page * PAGE_BLK; };
    if constexpr (!I8) {
        if (values) {
            if (page < 0) return;  // (the keys' workgroup says so)
            // eight dimensions of the tokens of one octet of the block
            const int h0 = (slot - kv_slots) * RA_HEADS, heads = min(RA_HEADS, a.pool.n_kv - h0);
            for (int i = tid; i < heads * (HD / 8) * 4; i += RA_THREADS) {
                const int oct = i & 3, d = (i >> 2) % (HD / 8) * 8, h = h0 + i / (HD / 2);
                const int first = max(8 * oct - t0, 0), last = min(8 * oct + 8 - t0, n);  // new tokens first .. last - 1
                if (first >= last) continue;
                const T* src = (const T*)a.v + r0 * a.v_ld + (long long)h * HD + d;
                C* dst = (C*)a.pool.v + block_of(h) * HD + d * PAGE_BLK + 8 * oct;
                uint32_t w[8][4];  // token j: its eight values
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int t = 8 * oct + j - t0;
                    const vec8<T> x = t >= first && t < last ? load8(src + t * a.v_ld) : vec8<T>{};
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        w[j][e] = (uint32_t)__builtin_bit_cast(uint16_t, (C)x[2 * e]) | (uint32_t)__builtin_bit_cast(uint16_t, (C)x[2 * e + 1]) << 16;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    uint32_t o[4];  // dimension e: its eight tokens
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        o[j] = __builtin_amdgcn_perm(w[2 * j + 1][e >> 1], w[2 * j][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
                    if (last - first == 8) {
                        *(uint4*)(dst + e * PAGE_BLK) = uint4{o[0], o[1], o[2], o[3]};
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const int t = 8 * oct + j - t0;
                            if (t >= first && t < last) ((uint16_t*)dst)[e * PAGE_BLK + j] = (uint16_t)(o[j >> 1] >> (16 * (j & 1)));
                        }
                    }
                }
            }
            return;
        }
    }
    // units of this workgroup's rows: source, its row stride and heads
    const int h0 = keys ? (I8 ? slot : slot * RA_HEADS) : (slot - kv_slots - v_slots) * (2 * RA_HEADS);
    const int heads = keys ? (I8 ? 1 : min(RA_HEADS, a.pool.n_kv - h0)) : min(2 * RA_HEADS, a.n_heads - h0);
    const long long ld = keys ? a.k_ld : a.q_ld;
    const T* src = (const T*)(keys ? a.k : a.q) + r0 * ld + h0 * HD;
    const int total = n * heads * un.all;
    const uint32_t by_units = ((1u << 20) + un.all - 1) / un.all;  // i / units as a product: i < 4096, units <= 16
    struct Batch {
        Piece2<T> p[RA_AHEAD];
        int u[RA_AHEAD], h[RA_AHEAD], t[RA_AHEAD];
    };
    auto fetch = [&](int i0) __attribute__((always_inline)) {
        Batch f;
#pragma unroll
        for (int k = 0; k < RA_AHEAD; k++) {
            const int i = i0 + k * RA_THREADS;
            const int th = (int)(((uint32_t)i * by_units) >> 20);
            f.u[k] = i - th * un.all;
            f.t[k] = (int)((uint32_t)th / (uint32_t)heads);
            f.h[k] = th - f.t[k] * heads;
            f.p[k] = i < total ? unit_load(src + f.t[k] * ld + f.h[k] * HD, f.u[k], un) : Piece2<T>{};
        }
        return f;
    };
    Batch f = fetch(tid);  // on its way while the angles are made
    for (int i = tid; i < n * half; i += RA_THREADS) {
        const int t = i / half, j = i - t * half;
        const double turns = (double)(p0 + t) * (a.inv_freq[j] * 0.15915494309189533577);
        float sn, cn;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cn);
        s_cs[i] = float2_t{cn * a.attn, sn * a.attn};
    }
    __syncthreads();
    auto turn_rows = [&](auto put) __attribute__((always_inline)) {
        for (int i0 = tid; i0 < total;) {
#pragma unroll
            for (int k = 0; k < RA_AHEAD; k++)
                if (i0 + k * RA_THREADS < total)
                    unit_turn(f.p[k], f.u[k], un, s_cs + f.t[k] * half, [&](int d, float8_t x) { put(f.t[k], f.h[k], d, x); });
            i0 += RA_AHEAD * RA_THREADS;
            if (i0 < total) f = fetch(i0);
        }
    };
    if (!keys) {
        T* dst = (T*)a.q_out + r0 * a.q_out_ld + h0 * HD;
        turn_rows([&](int t, int h, int d, float8_t x) { store8(dst + t * a.q_out_ld + h * HD + d, x); });
        return;
    }
    if (page < 0) {
        if (a.bt.status && tid == 0) atomicOr(&a.bt.status[b], PAGE_SEQ_BAD_PAGE);
        return;
    }
    if constexpr (!I8) {
        turn_rows([&](int t, int h, int d, float8_t x) {
            store8((C*)a.pool.k + block_of(h0 + h) * HD + page_k_at(t0 + t, d, HD, false), x);
        });
    } else {
        const int h = h0;
        const size_t at = block_of(h);
        turn_rows([&](int t, int, int d, float8_t x) { store8(s_k + t * LDK + d, x); });
        for (int i = tid; i < n * (HD / 8); i += RA_THREADS) {
            const int d = i % (HD / 8) * 8, t = i / (HD / 8);
            store8(s_v + t * LDK + d, __builtin_convertvector(load8((const T*)a.v + (r0 + t) * a.v_ld + (long long)h * HD + d), float8_t));
        }
        __syncthreads();
        // absmax scale of a (token, kv head): code = x / scale from the f32 scale, kept as fp16
        for (int row = tid >> 6; row < 2 * n; row += RA_THREADS / 64) {
            const float* src = (row & 1 ? s_v : s_k) + (row >> 1) * LDK;
            float m = fabsf(src[tid & 63]);
            if (HD == 128) m = fmaxf(m, fabsf(src[64 + (tid & 63)]));
            m = wave_max_f32(m);
            const float sc = m <= FLT_EPSILON ? 1.0f : m / 127.0f;
            if ((tid & 63) == 0) {
                s_sc[row & 1][row >> 1] = sc;
                (row & 1 ? a.pool.vs : a.pool.ks)[at + t0 + (row >> 1)] = __builtin_bit_cast(uint16_t, (_Float16)sc);
            }
        }
        __syncthreads();
        auto code = [](float x, float sc) { return (uint32_t)(uint8_t)(int8_t)fminf(fmaxf(roundf(x / sc), -127.0f), 127.0f); };
        for (int i = tid; i < n * (HD / 8); i += RA_THREADS) {
            const int d = i % (HD / 8) * 8, t = i / (HD / 8);
            uint2 w = {0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                w.x |= code(s_k[t * LDK + d + j], s_sc[0][t]) << (8 * j);
                w.y |= code(s_k[t * LDK + d + 4 + j], s_sc[0][t]) << (8 * j);
            }
            *(uint2*)((int8_t*)a.pool.k + at * HD + page_k_at(t0 + t, d, HD, true)) = w;
        }
        // values: one dimension's tokens of an octet
        for (int i = tid; i < HD * 4; i += RA_THREADS) {
            const int d = i % HD, oct = i / HD;
            const int first = max(8 * oct - t0, 0), last = min(8 * oct + 8 - t0, n);
            if (first >= last) continue;
            uint8_t* dst = (uint8_t*)a.pool.v + at * HD + page_v_at(8 * oct, d, HD, true);
            uint2 w = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int t = 8 * oct + j - t0;
                if (t < first || t >= last) continue;
                const uint32_t c = code(s_v[t * LDK + d], s_sc[1][t]);
                if (last - first < 8) dst[j] = (uint8_t)c;
                (j < 4 ? w.x : w.y) |= c << (8 * (j & 3));
            }
            if (last - first == 8) *(uint2*)dst = w;
        }
    }
}

template <typename T, int KVF>
int launch_rope_hd(const RopeAppendArgs& a, hipStream_t stream) {
    const int blocks = (a.bt.max_rows + 30) / PAGE_BLK + 1;  // blocks that max_rows positions can touch
    const int kv_slots = KVF == KV_INT8 ? a.pool.n_kv : (a.pool.n_kv + RA_HEADS - 1) / RA_HEADS;
    const dim3 grid(blocks, (KVF == KV_INT8 ? 1 : 2) * kv_slots + (a.n_heads + 2 * RA_HEADS - 1) / (2 * RA_HEADS), a.bt.nseq);
    if (a.pool.hd == 128) hipLaunchKernelGGL((rope_append_kernel<T, KVF, 128>), grid, dim3(RA_THREADS), 0, stream, a, kv_slots);
    else hipLaunchKernelGGL((rope_append_kernel<T, KVF, 64>), grid, dim3(RA_THREADS), 0, stream, a, kv_slots);
    return note_error(hipGetLastError());
}

}  // namespace

int launch_rope_append(const RopeAppendArgs& a, hipStream_t stream) {
    if (a.act == ACT_F32)
        return a.pool.fmt == KV_INT8 ? launch_rope_hd<float, KV_INT8>(a, stream) : launch_rope_hd<float, KV_F16>(a, stream);
    if (a.act == ACT_F16)
        return a.pool.fmt == KV_INT8 ? launch_rope_hd<_Float16, KV_INT8>(a, stream) : launch_rope_hd<_Float16, KV_F16>(a, stream);
    return launch_rope_hd<__bf16, KV_BF16>(a, stream);
}

}  // namespace aarh
