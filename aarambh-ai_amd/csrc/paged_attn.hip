// Attention of a call's new rows over the paged key / value cache.
//
// Rows of one sequence that read one kv head (its `group` query heads, token by token: row r is query head
// r % group of new token r / group) form the columns of S^T = K Q^T and O^T = V^T P^T.  In the matrix instructions'
// result layout a lane then holds the scores of ONE query for eight consecutive tokens, which is
// the operand layout of P^T: the softmax needs no exchange but a maximum over the four 16-lane
// rows of the wave, P never leaves the registers, and O's columns take the running factor lane by lane.
// The pages store K and V in operand order, so a wave's load is 1 KiB of consecutive bytes.
//
// Running maximum, sum and O are f32.  P is rounded to the pool's 16 bits for the product with V
// (2^-11 or 2^-8 of each weight, as V itself was); f32 queries are split into fp16 hi + lo
// halves, and so is P (2^-22 together): two matrix instructions in place of one.
//
// Few rows (paged_decode_kernel): bound by the cache's bytes, one pass, the cache split over the compute units and joined
// by a second launch; in short calls by that chain of launches and loads.  Many rows (paged_prompt_kernel): bound by the matrix
// instructions at the clock that the power budget leaves (fp16 runs 6% slower than bf16 with the same instructions).
// Measured, 32 query heads on 8 of size 128: one token over 4096 fp16 10 us (two launches); 16 tokens over 32768 bf16
// 258 us (6.4 TB/s); 32 x 4 rows over 4096 INT8, f32, 51 us (4.1 TB/s); 8192 rows bf16 552 us (1.0 PFLOP/s), with a cap and
// a window of 4096 532 us; 500 rows behind 3000 fp16 58 us.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "device_common.hpp"
#include "paged.hpp"

namespace aarh {

namespace {

typedef __bf16 bfrag_t __attribute__((ext_vector_type(8)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

constexpr float PA_LOG2E = 1.4426950408889634f;

// Element type of the matrix instructions for a pool format.
template <int KVF>
struct Mat {
    typedef typename std::conditional<KVF == KV_BF16, bfrag_t, half8_t>::type frag;
    typedef typename std::conditional<KVF == KV_BF16, __bf16, _Float16>::type elem;
    // The running reference of a column's exponents follows its maximum only when that is past it by
    // P_LAG (in powers of two), so most blocks leave O as it is.  fp16 weights are scaled by 2^P_BITS (cancelled by the sum):
    // the largest lies between 2^11 and 2^15, and the smallest steps of fp16 are 2^-35 of it.
    static constexpr float P_LAG = 4.f;
    static constexpr float P_BITS = KVF == KV_BF16 ? 0.f : 11.f;
};

template <int KVF>
__device__ __forceinline__ float4_t mfma16(typename Mat<KVF>::frag a, typename Mat<KVF>::frag b, float4_t c) {
    if constexpr (KVF == KV_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 8 INT8 codes as fp16, exactly: code + 128 in the mantissa of 1024, minus 1152
__device__ __forceinline__ half8_t i8_to_half8(uint32_t d0, uint32_t d1) {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    const half2v off = {(_Float16)1152.f, (_Float16)1152.f};
    d0 ^= 0x80808080u;
    d1 ^= 0x80808080u;
    union {
        half8_t h;
        half2v p[4];
    } r;
    r.p[0] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, d0, 0x04010400u)) - off;
    r.p[1] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, d0, 0x04030402u)) - off;
    r.p[2] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, d1, 0x04010400u)) - off;
    r.p[3] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, d1, 0x04030402u)) - off;
    return r.h;
}

__device__ __forceinline__ float row16_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row16_sum(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// tanh(x) = 1 - 2 / (exp(2 x) + 1).  Near zero that is off by 2^-23 absolutely, which a score of 16-bit
// operands does not notice; PRECISE takes the series there.
template <bool PRECISE>
__device__ __forceinline__ float tanh_f32(float x) {
    const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * (2.f * PA_LOG2E)) + 1.f);
    if constexpr (!PRECISE) return big;
    const float y2 = x * x;
    const float series = x * (1.f + y2 * (-0.33333333333f + y2 * (0.13333333333f + y2 * (-0.053968253968f + y2 * (0.021869488536f - y2 * 0.0088632355299f)))));
    return fabsf(x) < 0.3f ? series : big;
}

// What a tile of query rows needs to know of its sequence.
struct TileInfo {
    PageSeq s;
    int b, kvh, r0;        // first row (token x group member) of the tile
    int p_lo, p_hi, pre;   // positions of its first and last rows; prefix length
    int low;               // first key that the window leaves to any row
    int pre_blk, lo_blk, n;  // 32-token blocks it visits: 0 .. pre_blk - 1, then lo_blk ..; n in all
};

// Blocks of a tile: those of the prefix that lie before the window, then from the window's start to
// the last visible key.
__device__ __forceinline__ bool tile_info(const PagedAttnArgs& a, int b, int kvh, int tile, int tile_rows, int group, TileInfo* t) {
    if (!page_seq(a.bt.row_off, a.bt.kv_len, b, a.bt.rows, a.bt.max_rows, a.bt.max_kv, &t->s)) {
        if (a.bt.status && threadIdx.x == 0) atomicOr(&a.bt.status[b], PAGE_SEQ_BAD_LENGTH);
        return false;
    }
    t->b = b;
    t->kvh = kvh;
    t->r0 = tile * tile_rows;
    const int rows = t->s.rows * group;
    if (t->r0 >= rows) return false;
    const int pos0 = t->s.kv_len - t->s.rows;
    t->p_lo = pos0 + t->r0 / group;
    t->p_hi = pos0 + (min(t->r0 + tile_rows, rows) - 1) / group;
    t->pre = a.prefix ? min(max(a.prefix[b], 0), t->s.kv_len) : 0;
    t->low = a.window ? max(0, t->p_lo - a.window + 1) : 0;
    t->lo_blk = t->low >> 5;
    t->pre_blk = min((t->pre + 31) >> 5, t->lo_blk);
    t->n = t->pre_blk + ((max(t->p_hi + 1, t->pre) + 31) >> 5) - t->lo_blk;
    return true;
}

// Tokens base .. base + n - 1 as bits: those from low to high, and those before pre.
__device__ __forceinline__ uint32_t seen_bits(int base, int low, int high, int pre, int n) {
    auto ones = [](int k) { return k >= 32 ? 0xFFFFFFFFu : (1u << k) - 1u; };
    auto upto = [&](int t) { return ones(min(max(t - base, 0), n)); };
    return (upto(high + 1) & ~upto(low)) | upto(pre);
}
// 16-bit masks of eight tokens (bits of b)
__device__ __forceinline__ u32x4_t keep_words(uint32_t b) {
    u32x4_t k;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t lo = (uint32_t)((int32_t)(b << (31 - 2 * i)) >> 31), hi = (uint32_t)((int32_t)(b << (30 - 2 * i)) >> 31);
        k[i] = (lo & 0xFFFFu) | (hi & 0xFFFF0000u);
    }
    return k;
}

// Values that are not finite.  In a product they would also reach the rows that do not see their token (0 x inf), so where rows of
// a tile see different tokens of a block such values are taken out of V and counted for the rows that do see them.
template <int KVF>
struct Odd {
    static constexpr bool BF = KVF == KV_BF16;
    static constexpr uint32_t INF = BF ? 0x7F80u : 0x7C00u, ONE = BF ? 0x3F80u : 0x3C00u, C64 = BF ? 0x4280u : 0x5400u, C4096 = BF ? 0x4580u : 0x6C00u;
    typedef typename Mat<KVF>::frag frag;
    typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
    // largest magnitude of both halves
    static __device__ __forceinline__ uint32_t top(u32x4_t w, uint32_t t) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            t = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, w[i] & 0x7FFF7FFFu), __builtin_bit_cast(u16x2_t, t)));
        return t;
    }
    static __device__ __forceinline__ bool any(uint32_t t) { return __any((t & 0xFFFFu) >= INF || t >> 16 >= INF); }
    // marks to be counted: 1 for +inf, 64 for -inf, 4096 for NaN (a block has 32 tokens)
    static __device__ __forceinline__ frag marks(u32x4_t w) {
        auto mark = [](uint32_t h) {
            const uint32_t m = h & 0x7FFFu;
            return m < INF ? 0u : m > INF ? C4096 : h == INF ? ONE : C64;
        };
        u32x4_t r;
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = mark(w[i] & 0xFFFFu) | mark(w[i] >> 16) << 16;
        return __builtin_bit_cast(frag, r);
    }
    static __device__ __forceinline__ u32x4_t finite(u32x4_t w) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] &= ((w[i] & 0x7FFFu) >= INF ? 0u : 0xFFFFu) | ((w[i] >> 16 & 0x7FFFu) >= INF ? 0u : 0xFFFF0000u);
        return w;
    }
    // eight tokens' visibility as an operand
    static __device__ __forceinline__ frag seen(uint32_t bits) { return __builtin_bit_cast(frag, keep_words(bits) & (ONE | ONE << 16)); }
    // what the sum of the marks that a row sees adds to its result
    static __device__ __forceinline__ float worth(float marks) {
        const int n = (int)marks;
        return (n & 63 ? INFINITY : 0.f) + (n >> 6 & 63 ? -INFINITY : 0.f) + (n >> 12 ? NAN : 0.f);
    }
};

// Workgroup -> pair of sequence and kv head (fastest), tile of its rows, split of its keys.  Workgroups go to the
// eight dies in turn, so tiles of a pair, which read the same blocks, share a die's cache when there are 8 n pairs.
struct Place {
    int pair, tile, split;
};
__device__ __forceinline__ Place place_of(const PagedAttnArgs& a, int tiles) {
    const int pairs = a.bt.nseq * a.pool.n_kv, rest = blockIdx.x / pairs;
    return {(int)blockIdx.x - rest * pairs, rest % tiles, rest / tiles};
}

__device__ __forceinline__ int tile_block(const TileInfo& t, int k) { return k < t.pre_blk ? k : t.lo_blk + (k - t.pre_blk); }

__device__ __forceinline__ int head_of(const PagedAttnArgs& a, int kvh, int m, int group) {
    return a.grouped ? kvh * group + m : m * a.pool.n_kv + kvh;
}

// Workspace of a call split over the keys: [split][row x head][hd] weighted sums, then their (maximum, sum).
__device__ __forceinline__ float* part_o(const PagedAttnArgs& a, int split, long long slot) {
    return (float*)a.workspace + ((long long)split * a.bt.rows * a.n_heads + slot) * a.pool.hd;
}
__device__ __forceinline__ float2_t* part_ml(const PagedAttnArgs& a, int splits, int split, long long slot) {
    const long long slots = (long long)a.bt.rows * a.n_heads;
    return (float2_t*)((float*)a.workspace + splits * slots * a.pool.hd) + split * slots + slot;
}

// ---------------------------------------------------------------------------
// Few rows: the cache is streamed through the registers
// ---------------------------------------------------------------------------
// Waves of a workgroup, which share its blocks one by one.  INT8 blocks need more arithmetic for their bytes, and a second
// wave on each SIMD (32 x 4 rows over 4096 tokens 52 us, 76 with four waves); 16-bit pools stream as
// well with four (64 x 1 over 4096 6.3 TB/s either way) and have less to join.
constexpr int dc_waves(int kvf) { return kvf == KV_INT8 ? 8 : 4; }

template <typename T, int KVF, int HD, int NT, bool ONCE>
__global__ __launch_bounds__(dc_waves(KVF) * 64) void paged_decode_kernel(PagedAttnArgs a, int group, int tiles, int splits, int per) {
    typedef typename Mat<KVF>::frag frag;
    typedef typename Mat<KVF>::elem elem;
    constexpr bool I8 = KVF == KV_INT8, F32 = std::is_same<T, float>::value;
    constexpr int KS = HD / 32;              // k-steps of K Q^T
    constexpr int DT = HD / 16;              // 16-dimension tiles of O^T
    constexpr int KL = I8 ? HD / 32 : HD / 16;  // 16-byte pieces of a lane's share of a K (or V) block
    constexpr int BLK = PAGE_BLK * HD * (I8 ? 1 : 2);
    constexpr int LDO = HD + 4;
    constexpr int DC_WAVES = dc_waves(KVF);
    __shared__ float s_o[DC_WAVES][16 * LDO];
    __shared__ float2_t s_ml[DC_WAVES][16];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, lg = lane >> 4;
    const Place at = place_of(a, tiles);
    const int split = at.split;
    TileInfo t;
    if (!tile_info(a, at.pair / a.pool.n_kv, at.pair % a.pool.n_kv, at.tile, 16 * NT, group, &t)) return;
    const int k0 = split * per, k1 = min(k0 + per, t.n);
    const int rows = t.s.rows * group, pos0 = t.s.kv_len - t.s.rows;

    // this lane's queries: columns lr of NT tiles
    frag qh[NT][KS], ql[NT][F32 ? KS : 1];
    float qs[NT], slope[NT];
    int pos[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int r = t.r0 + nt * 16 + lr, rr = min(r, rows - 1), tok = rr / group;
        const int h = head_of(a, t.kvh, rr - tok * group, group);
        pos[nt] = r < rows ? pos0 + tok : -1;  // -1: a column of no row, sees at most prefix keys
        slope[nt] = a.slopes ? a.slopes[h] * PA_LOG2E : 0.f;
        const T* q = (const T*)a.q + (long long)(t.s.row0 + tok) * a.q_ld + (long long)h * HD + 16 * lg;
        qs[nt] = fabsf(a.scale);
        if constexpr (F32) {
            float x[KS][8], top = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float* src = q + 64 * (ks >> 1) + 8 * (ks & 1);
                const float4_t u = *(const float4_t*)src, v = *(const float4_t*)(src + 4);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[ks][j] = u[j];
                    x[ks][4 + j] = v[j];
                }
#pragma unroll
                for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[ks][j]));
            }
            // a power of two brings the row's largest value to [1/2, 1) (fp16's range); the scale takes it back
            const int e = __builtin_amdgcn_frexp_expf(row16_max(top));
            const float inv = ldexpf(1.f, -max(e, -120));
            qs[nt] = ldexpf(qs[nt], max(e, -120));
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float v = x[ks][j] * inv;
                    qh[nt][ks][j] = (_Float16)v;
                    ql[nt][ks][j] = (_Float16)(v - (float)qh[nt][ks][j]);
                }
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                if constexpr (std::is_same<T, elem>::value) qh[nt][ks] = *(const frag*)(q + 64 * (ks >> 1) + 8 * (ks & 1));
            }
        }
        if (a.scale < 0.f) {  // a negative scale's sign goes to the query, so that the largest product is the largest score
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                qh[nt][ks] = -qh[nt][ks];
                if constexpr (F32) ql[nt][ks] = -ql[nt][ks];
            }
        }
        qs[nt] = fmaxf(qs[nt], 1e-30f);  // -inf of a masked key stays what it is
    }

    float m[NT], l[NT];
    float4_t o[NT][DT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m[nt] = -INFINITY;
        l[nt] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[nt][d] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

    const int32_t* table = a.bt.tables + t.b * a.bt.table_ld;
    const int shift = a.pool.page_shift - 5;  // blocks of a page
    const bool plain = a.softcap == 0.f && a.slopes == nullptr;
    const float inv_cap = a.softcap > 0.f ? 1.f / a.softcap : 0.f;
    u32x4_t kr[KL], vr[KL], ksc, vsc;
    // this wave's blocks: k0 + wid, k0 + wid + DC_WAVES, ..
    auto page_at = [&](int k) __attribute__((always_inline)) {
        const int blk = tile_block(t, k);
        return table[blk >> shift];
    };
    size_t off = 0;  // element offset of the block in K and V
    auto locate = [&](int k, int page) __attribute__((always_inline)) {
        const int blk = tile_block(t, k);
        const int p = page >= 0 && page < a.pool.n_pages ? page : 0;
        off = ((((size_t)p * a.pool.n_kv + t.kvh) << shift) + (blk & ((1 << shift) - 1))) * PAGE_BLK;
    };
    // ONCE: a block that no other workgroup reads does not stay in the caches
    auto load_block = [&](u32x4_t(&r)[KL], const char* p) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KL; i++) {
            if constexpr (ONCE) r[i] = __builtin_nontemporal_load((const u32x4_t*)(p + i * 1024));
            else r[i] = *(const u32x4_t*)(p + i * 1024);
        }
    };
    auto load_k = [&]() __attribute__((always_inline)) {
        load_block(kr, (const char*)a.pool.k + off * (BLK / PAGE_BLK) + lane * 16);
        if constexpr (I8) ksc = *(const u32x4_t*)(a.pool.ks + off + 8 * lg);
    };
    auto load_v = [&]() __attribute__((always_inline)) {
        load_block(vr, (const char*)a.pool.v + off * (BLK / PAGE_BLK) + (I8 ? lane : lr * 4 + lg) * 16);
        if constexpr (I8) vsc = *(const u32x4_t*)(a.pool.vs + off + 8 * lg);
    };
    auto sc_at = [](u32x4_t s, int i) __attribute__((always_inline)) {
        const uint32_t w = s[i >> 1];
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w >> 16 : w & 0xFFFFu));
    };
    bool bad = false;
    int k = k0 + wid;
    int page = 0, page_next = 0;
    if (k < k1) {
        page = page_at(k);
        page_next = page_at(min(k + DC_WAVES, k1 - 1));
        locate(k, page);
        load_k();
        load_v();
    }
    for (; k < k1; k += DC_WAVES) {
        const int t0 = tile_block(t, k) * PAGE_BLK;
        const bool absent = page < 0 || page >= a.pool.n_pages;
        bad |= absent;
        const int kn = k + DC_WAVES;
        // scores: S^T of tokens 8 lg + 4 ts + i
        float4_t s[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) s[nt][0] = s[nt][1] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ts = 0; ts < 2; ts++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                frag ka;
                if constexpr (I8) {
                    const u32x4_t w = kr[ts * (KS / 2) + (ks >> 1)];
                    ka = ks & 1 ? i8_to_half8(w[2], w[3]) : i8_to_half8(w[0], w[1]);
                } else {
                    ka = __builtin_bit_cast(frag, kr[ts * KS + ks]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    s[nt][ts] = mfma16<KVF>(ka, qh[nt][ks], s[nt][ts]);
                    if constexpr (F32) s[nt][ts] = mfma16<KVF>(ka, ql[nt][ks], s[nt][ts]);
                }
            }
        const u32x4_t ksc_now = ksc;
        if (kn < k1) {
            locate(kn, page_next);
            load_k();
        }
        // visible to every row of the tile: no masks
        const bool whole = !absent && t0 + PAGE_BLK - 1 <= t.p_lo && (a.window == 0 || t0 > t.p_hi - a.window || t0 + PAGE_BLK <= t.pre);
        float vexp = 0.f;
        if constexpr (I8) {
            // INT8: a weight is multiplied by its token's V scale before it is rounded to fp16, so
            // the reference of the exponents rises by the exponent of the block's largest scale
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int tok = t0 + 8 * lg + i;
                const float v = sc_at(vsc, i);
                top = fmaxf(top, tok <= t.p_hi || tok < t.pre ? v : 0.f);
            }
            top = row16_max(top);
            vexp = top > 0x1p-20f ? (float)__builtin_amdgcn_frexp_expf(top) : -20.f;
        }
        frag ph[NT], pl[F32 ? NT : 1];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = s[nt][i >> 2][i & 3];
                if constexpr (I8) x[i] *= sc_at(ksc_now, i);
            }
            float c = qs[nt] * PA_LOG2E;
            if (!plain) {
                const float from = slope[nt] * (float)(t0 + 8 * lg - pos[nt]);
                if (a.softcap > 0.f) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = a.softcap * tanh_f32<F32>(x[i] * qs[nt] * inv_cap);
                    c = PA_LOG2E;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = fmaf(x[i], c, fmaf(slope[nt], (float)i, from));
                c = 1.f;
            }
            if (!whole) {
                const uint32_t seen = absent ? 0u : seen_bits(t0 + 8 * lg, a.window ? max(0, pos[nt] - a.window + 1) : 0, pos[nt], t.pre, 8);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = (seen >> i) & 1u ? x[i] : -INFINITY;
            }
            float mx = x[0];
#pragma unroll
            for (int i = 1; i < 8; i++) mx = fmaxf(mx, x[i]);
            mx = row16_max(mx) * c;
            if constexpr (I8) mx += vexp;
            if (__any(mx > m[nt] + Mat<KVF>::P_LAG)) {
                const float mn = fmaxf(m[nt], mx);
                const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[nt] - mn);
                l[nt] *= alpha;
#pragma unroll
                for (int d = 0; d < DT; d++) o[nt][d] *= alpha;
                m[nt] = mn;
            }
            const float ref = (m[nt] == -INFINITY ? 0.f : m[nt]) - Mat<KVF>::P_BITS;
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                p[i] = __builtin_amdgcn_exp2f(fmaf(x[i], c, -ref));
                l[nt] += p[i];
                if constexpr (I8) p[i] = p[i] == 0.f ? 0.f : p[i] * sc_at(vsc, i);  // a token that is not there may have any scale
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                ph[nt][i] = (elem)p[i];
                if constexpr (F32) pl[nt][i] = (elem)(p[i] - (float)ph[nt][i]);
            }
        }
        // tokens that no row sees may hold anything, also NaN: their V is taken as zero
        if constexpr (!I8) {
            if (!whole) {
                const u32x4_t keep = keep_words(absent ? 0u : seen_bits(t0 + 8 * lg, t.low, t.p_hi, t.pre, 8));
#pragma unroll
                for (int i = 0; i < KL; i++) vr[i] &= keep;
                if (t.p_lo < t.p_hi && t0 + PAGE_BLK > t.pre) {
                    uint32_t top = 0;
#pragma unroll
                    for (int i = 0; i < KL; i++) top = Odd<KVF>::top(vr[i], top);
                    if (__builtin_expect(Odd<KVF>::any(top), 0)) {
                        frag seen[NT];
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
                            seen[nt] = Odd<KVF>::seen(absent ? 0u : seen_bits(t0 + 8 * lg, a.window ? max(0, pos[nt] - a.window + 1) : 0, pos[nt], t.pre, 8));
#pragma unroll
                        for (int d = 0; d < DT; d++) {
                            const frag marks = Odd<KVF>::marks(vr[d]);
                            vr[d] = Odd<KVF>::finite(vr[d]);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                const float4_t c = mfma16<KVF>(marks, seen[nt], float4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                                for (int i = 0; i < 4; i++) o[nt][d][i] += Odd<KVF>::worth(c[i]);
                            }
                            __builtin_amdgcn_sched_barrier(0);  // (one at a time: few registers)
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            frag va;
            if constexpr (I8) {
                const u32x4_t w = vr[d >> 1];
                va = d & 1 ? i8_to_half8(w[2], w[3]) : i8_to_half8(w[0], w[1]);
            } else {
                va = __builtin_bit_cast(frag, vr[d]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                o[nt][d] = mfma16<KVF>(va, ph[nt], o[nt][d]);
                if constexpr (F32) o[nt][d] = mfma16<KVF>(va, pl[nt], o[nt][d]);
            }
        }
        if (kn < k1) {
            load_v();
            page = page_next;
            page_next = page_at(min(kn + DC_WAVES, k1 - 1));
        }
    }
    if (bad && a.bt.status && lane == 0) atomicOr(&a.bt.status[t.b], PAGE_SEQ_BAD_PAGE);

    // the waves' shares of each column: joined through LDS
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const float lsum = row16_sum(l[nt]);
        if (nt) __syncthreads();
        if (lane < 16) s_ml[wid][lr] = float2_t{m[nt], lsum};
#pragma unroll
        for (int d = 0; d < DT; d++) *(float4_t*)&s_o[wid][lr * LDO + 16 * d + 4 * lg] = o[nt][d];
        __syncthreads();
        for (int i = tid; i < 16 * (HD / 4); i += DC_WAVES * 64) {
            const int c = i / (HD / 4), d = i % (HD / 4) * 4;
            const int r = t.r0 + nt * 16 + c;
            if (r >= rows) continue;
            float M = s_ml[0][c][0];
#pragma unroll
            for (int w = 1; w < DC_WAVES; w++) M = fmaxf(M, s_ml[w][c][0]);
            float L = 0.f;
            float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < DC_WAVES; w++) {
                const float2_t ml = s_ml[w][c];
                const float f = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - M);
                L += ml[1] * f;
                acc += *(const float4_t*)&s_o[w][c * LDO + d] * f;
            }
            const int tok = r / group, h = head_of(a, t.kvh, r - tok * group, group);
            if (splits > 1) {
                const long long slot = (long long)(t.s.row0 + tok) * a.n_heads + h;
                *(float4_t*)(part_o(a, split, slot) + d) = acc;
                if (d == 0) *part_ml(a, splits, split, slot) = float2_t{M, L};
            } else {
                const float inv = L > 0.f ? 1.f / L : 0.f;
                typedef T out4 __attribute__((ext_vector_type(4)));
                *(out4*)((T*)a.out + (long long)(t.s.row0 + tok) * a.out_ld + (long long)h * HD + d) =
                    out4{(T)(acc[0] * inv), (T)(acc[1] * inv), (T)(acc[2] * inv), (T)(acc[3] * inv)};
            }
        }
    }
}

// Joins the splits of a call.  HD / 4 lanes take one split's sums of a (row, head) at a time, so a wave has PAR = 2 (HD 128)
// or 4 splits in hand at once.  Bound by the latency of its loads, so many of a wave's are under way together: WAVES waves a slot
// (a (row, head)) where there are few slots and many splits, SLOTS slots a wave where there are many slots and few splits.
template <typename T, int HD, int SLOTS, int WAVES>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs a, int splits) {
    constexpr int LN = HD / 4, PAR = 64 / LN, SPAN = 64 / SLOTS, AHEAD = SLOTS > 1 ? 2 : 8, STRIDE = PAR * WAVES;
    const int b = blockIdx.y, lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = lane % LN * 4;
    PageSeq s;
    if (!page_seq(a.bt.row_off, a.bt.kv_len, b, a.bt.rows, a.bt.max_rows, a.bt.max_kv, &s)) return;
    const long long at = ((long long)blockIdx.x * (4 / WAVES) + wid / WAVES) * SLOTS, all = (long long)s.rows * a.n_heads;
    if (at >= all) return;  // (WAVES 4: the whole workgroup)
    const long long slot = (long long)s.row0 * a.n_heads + at;
    const int k0 = wid % WAVES * PAR + lane / LN;  // splits k0, k0 + STRIDE, ..
    float4_t v[SLOTS][AHEAD];
    auto load = [&](int from) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < SLOTS; r++)
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int k = from + i * STRIDE;
                v[r][i] = k < splits && at + r < all ? *(const float4_t*)(part_o(a, k, slot + r) + d) : float4_t{0.f, 0.f, 0.f, 0.f};
            }
    };
    load(k0);
    float2_t ml = {-INFINITY, 0.f};  // lane SPAN r + k: split k of slot r
    if (lane % SPAN < splits && at + lane / SPAN < all) ml = *part_ml(a, splits, lane % SPAN, slot + lane / SPAN);
    float M = ml[0];
#pragma unroll
    for (int x = 1; x < SPAN; x *= 2) M = fmaxf(M, __shfl_xor(M, x));
    const float f = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - M);
    float L = ml[1] * f;
#pragma unroll
    for (int x = 1; x < SPAN; x *= 2) L += __shfl_xor(L, x);
    float4_t acc[SLOTS] = {};
    for (int from = 0;;) {
#pragma unroll
        for (int r = 0; r < SLOTS; r++)
#pragma unroll
            for (int i = 0; i < AHEAD; i++) acc[r] += v[r][i] * __shfl(f, r * SPAN + ((from + k0 + i * STRIDE) & (SPAN - 1)));
        from += AHEAD * STRIDE;
        if (SLOTS > 1 || from >= splits) break;
        load(from + k0);
    }
#pragma unroll
    for (int r = 0; r < SLOTS; r++)
#pragma unroll
        for (int x = LN; x < 64; x *= 2)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[r][j] += __shfl_xor(acc[r][j], x);
    if constexpr (WAVES > 1) {
        __shared__ float4_t s_acc[WAVES - 1][LN];
        if (wid && lane < LN) s_acc[wid - 1][lane] = acc[0];
        __syncthreads();
        if (wid || lane >= LN) return;
#pragma unroll
        for (int w = 0; w < WAVES - 1; w++) acc[0] += s_acc[w][lane];
    }
#pragma unroll
    for (int r = 0; r < SLOTS; r++) {
        const float Lr = __shfl(L, r * SPAN);
        if (lane / LN != r % PAR || at + r >= all) continue;  // every part of the wave has the sums
        const float inv = Lr > 0.f ? 1.f / Lr : 0.f;
        typedef T out4 __attribute__((ext_vector_type(4)));
        *(out4*)((T*)a.out + (s.row0 + (at + r) / a.n_heads) * a.out_ld + ((at + r) % a.n_heads) * HD + d) =
            out4{(T)(acc[r][0] * inv), (T)(acc[r][1] * inv), (T)(acc[r][2] * inv), (T)(acc[r][3] * inv)};
    }
}

// ---------------------------------------------------------------------------
// Many rows: tiles of 128 rows share each block through LDS
//
// Four waves of 32 columns each (32 x 32 matrix instructions: an operand read from LDS serves 32 queries). 64 tokens a
// step, two steps' pages in LDS: the next step's loads go straight to LDS while this one is computed.
// V^T pieces are placed so that the lanes of a read (consecutive dimensions, one token octet) fall on
// different banks: piece (dimension d, octet q) of a 16-dimension KiB sits at 4 d + (q ^ f(d)).
// ---------------------------------------------------------------------------
typedef float float16_t __attribute__((ext_vector_type(16)));

template <int KVF>
__device__ __forceinline__ float16_t mfma32(typename Mat<KVF>::frag a, typename Mat<KVF>::frag b, float16_t c) {
    if constexpr (KVF == KV_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float half_max(float x) {
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Piece i (of 4) of 1 KiB steps from a buffer offset to LDS: the instruction's offset counts for both sides, so four
// pieces share M0 and the scalar offset.
__device__ __forceinline__ void lds_piece(__amdgpu_buffer_rsrc_t r, const void* lds_dst, int voff, int soff, int i) {
    const unsigned base = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)lds_dst);
    switch (i) {
#define AARH_PIECE(N) asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen offset:%3 lds" ::"v"(voff), "s"(r), "s"(soff), "n"((N) * 1024), "{m0}"(base) : "memory")
        case 0: AARH_PIECE(0); break;
        case 1: AARH_PIECE(1); break;
        case 2: AARH_PIECE(2); break;
        default: AARH_PIECE(3); break;
#undef AARH_PIECE
    }
}

constexpr int PF_WAVES = 4, PF_ROWS = 32 * PF_WAVES;

// MODE 0: scores as they are, 1: capped, 2: a slope per head (capped or not)
template <typename T, int KVF, int HD, int MODE>
__global__ __launch_bounds__(PF_WAVES * 64, 2) void paged_prompt_kernel(PagedAttnArgs a, int group, int tiles, int splits, int per) {
    typedef typename Mat<KVF>::frag frag;
    typedef typename Mat<KVF>::elem elem;
    constexpr bool I8 = KVF == KV_INT8, F32 = std::is_same<T, float>::value;
    constexpr int KS = HD / 16;  // k-steps of K Q^T: (64-dimension part, half of 16, pair of lane groups)
    constexpr int DT = HD / 32;  // 32-dimension tiles of O^T
    constexpr int BLK = PAGE_BLK * HD * (I8 ? 1 : 2);
    constexpr int KIB = BLK / 1024;  // wave loads of a block of K (or V)
    __shared__ __attribute__((aligned(1024))) char pf_lds[8 * BLK];  // [2 stages][K: 2 blocks | V: 2 blocks]
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), hk = lane >> 5, m = lane & 31;
    const Place place = place_of(a, tiles);
    const int split = place.split;
    TileInfo t;  // the longest rows first
    if (!tile_info(a, place.pair / a.pool.n_kv, place.pair % a.pool.n_kv, tiles - 1 - place.tile, PF_ROWS, group, &t)) return;
    const int k0 = split * per, k1 = min(k0 + per, t.n);
    const int rows = t.s.rows * group, pos0 = t.s.kv_len - t.s.rows;

    // this lane's query
    // (columns past the last row repeat it, and are not stored)
    const int r = t.r0 + wid * 32 + m, rr = min(r, rows - 1), tok = rr / group;
    const int h = head_of(a, t.kvh, rr - tok * group, group);
    const int pos = pos0 + tok;
    const float slope = MODE == 2 ? a.slopes[h] * PA_LOG2E : 0.f;
    const int w_lo = pos0 + min(t.r0 + wid * 32, rows - 1) / group, w_hi = pos0 + min(t.r0 + wid * 32 + 31, rows - 1) / group;
    const bool idle = t.r0 + wid * 32 >= rows;  // a wave without rows
    frag qh[KS], ql[F32 ? KS : 1];
    float qs = fabsf(a.scale);
    {
        const T* q = (const T*)a.q + (long long)(t.s.row0 + tok) * a.q_ld + (long long)h * HD + 16 * hk;
        auto dim = [](int ks) { return 64 * (ks >> 2) + 32 * (ks & 1) + 8 * ((ks >> 1) & 1); };
        if constexpr (F32) {
            float x[KS][8], top = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float4_t u = *(const float4_t*)(q + dim(ks)), v = *(const float4_t*)(q + dim(ks) + 4);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[ks][j] = u[j];
                    x[ks][4 + j] = v[j];
                }
#pragma unroll
                for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[ks][j]));
            }
            const int e = max(__builtin_amdgcn_frexp_expf(half_max(top)), -120);
            const float inv = ldexpf(1.f, -e);
            qs = ldexpf(qs, e);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float v = x[ks][j] * inv;
                    qh[ks][j] = (_Float16)v;
                    ql[ks][j] = (_Float16)(v - (float)qh[ks][j]);
                }
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                if constexpr (std::is_same<T, elem>::value) qh[ks] = *(const frag*)(q + dim(ks));
            }
        }
        if (a.scale < 0.f) {  // a negative scale's sign goes to the query, so that the largest product is the largest score
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                qh[ks] = -qh[ks];
                if constexpr (F32) ql[ks] = -ql[ks];
            }
        }
        qs = fmaxf(qs, 1e-30f);  // -inf of a masked key stays what it is
    }

    const int32_t* table = a.bt.tables + t.b * a.bt.table_ld;
    const int shift = a.pool.page_shift - 5;
    const bool capped = a.softcap > 0.f;
    const float inv_cap = capped ? 1.f / a.softcap : 0.f, cap2 = a.softcap * PA_LOG2E;
    // lane's places in LDS: K token row (bits 2 and 3 of its number change places: see paged_rule.hpp), V piece
    const int k_lane = ((m >> 3) & 1) * (BLK / 2) + hk * 256 + (8 * (m >> 4) + 4 * ((m >> 2) & 1) + (m & 3)) * 16;
    auto swz = [](int d) { return ((d >> 1) & 3) ^ ((d >> 3) & 1); };
    const int v_lane = I8 ? hk * 256 + (m & 15) * 16 + (m >> 4) * 8 : (m >> 4) * 1024 + (m & 15) * 64 + ((hk ^ swz(m & 15)) << 4);
    const int v_src = I8 ? lane * 16 : ((lane & ~3) + ((lane & 3) ^ swz(lane >> 2))) * 16;  // global piece for LDS place `lane`

    // Blocks of a step, two: their numbers in the sequence and pages (wave-uniform).  A step's pages are read
    // a step before its loads are issued, and these a step before the data is needed.
    struct Step {
        int blk[2], page[2];
    };
    auto look_up = [&](int k) __attribute__((always_inline)) {
        Step s;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            s.blk[j] = tile_block(t, min(k + j, k1 - 1));
            s.page[j] = *(const int32_t*)((const char*)table + ((uint32_t)(s.blk[j] >> shift) << 2));
        }
        return s;
    };
    auto settle = [&](Step s) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int p = __builtin_amdgcn_readfirstlane(s.page[j]);
            s.page[j] = (unsigned)p < (unsigned)a.pool.n_pages ? p : -1;
        }
        return s;
    };
    // first token of a block in the pool's arrays of tokens
    auto token_of = [&](int blk, int page) __attribute__((always_inline)) {
        return ((((size_t)max(page, 0) * a.pool.n_kv + t.kvh) << shift) + (blk & ((1 << shift) - 1))) * PAGE_BLK;
    };
    // wave w loads the keys (w < 2) or values of block w % 2 of a step
    const int my_j = wid & 1, my_v = wid >> 1;
    const char* my_pool = (const char*)(my_v ? a.pool.v : a.pool.k);
    const int my_src = my_v ? v_src : lane * 16;
    // ... one KiB at a time: pieces of the next step's loads go between this step's products (issued in a row they
    // hold the wave until the address unit has taken them: 1000 cycles of a step)
    struct Load {
        uint32_t lo, hi;  // global address of the block
        char* dst;
    };
    auto load_of = [&](const Step& s, int buf) __attribute__((always_inline)) {
        const size_t at = my_j ? token_of(s.blk[1], s.page[1]) : token_of(s.blk[0], s.page[0]);
        const uint64_t p = (uint64_t)(my_pool + at * (BLK / PAGE_BLK));
        return Load{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)p), (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32)),
                    pf_lds + buf * (4 * BLK) + (2 * my_v + my_j) * BLK};
    };
    auto piece = [&](const Load& ld, int i) __attribute__((always_inline)) {
        lds_piece(coh_rsrc((const void*)(((uint64_t)ld.hi << 32) | ld.lo)), ld.dst + (i & ~3) * 1024, my_src, (i & ~3) * 1024, i & 3);
    };
    auto pieces = [&](const Load& ld) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KIB; i++) piece(ld, i);
    };

    float mx_run = -INFINITY, l = 0.f;
    float16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.f;
    const int wlow = a.window ? max(0, w_lo - a.window + 1) : 0;

    // A step of this wave in two parts.  MASK: the general form.  Without MASK every row of the tile sees every token.
    struct Work {
        float16_t s[2];             // scores, then weights
        float vsc[2][I8 ? 16 : 1];  // INT8: scales of V
        float mx;                   // largest exponent of the column
        bool skip[2];               // blocks that no row of this wave sees
    };
    auto factor = [&](auto mask) { return (!mask.value && MODE == 1) || MODE == 0 ? qs * PA_LOG2E : 1.f; };
    auto scores = [&](const Step& cur, int buf, bool two, const Load* ld, auto mask, Work& w) __attribute__((always_inline)) {
        constexpr bool MASK = mask.value;
        constexpr bool direct = !MASK && MODE == 1;
        const float c = factor(mask);
        float16_t(&s)[2] = w.s;
        auto& vsc = w.vsc;
        const int t0[2] = {cur.blk[0] * PAGE_BLK, cur.blk[1] * PAGE_BLK};
        w.skip[0] = w.skip[1] = false;
        if constexpr (MASK) {
#pragma unroll
            for (int j = 0; j < 2; j++)
                w.skip[j] = (j && !two) || cur.page[j] < 0 || (t0[j] >= t.pre && (t0[j] > w_hi || t0[j] + PAGE_BLK <= wlow));
            if (idle || (w.skip[0] && w.skip[1])) return false;
        }
        const char* kb = pf_lds + buf * (4 * BLK) + k_lane;
        s[0] = s[1] = float16_t{};
        // operands are read two iterations before their products
        constexpr int QN = I8 ? KS / 2 : KS;  // iterations; INT8 operands are two k-steps each
        static_assert(QN == KIB, "one piece of the next step an iteration");
        u32x4_t ka[3][2];
        auto read = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 2; j++) ka[i % 3][j] = *(const u32x4_t*)(kb + j * BLK + (i >> 1) * 1024 + (i & 1) * 512);
        };
        read(0);
        if (QN > 1) read(1);
#pragma unroll
        for (int i = 0; i < QN; i++) {
            if (i + 2 < QN) read(i + 2);
            if constexpr (!MASK) piece(*ld, i);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const u32x4_t kw = ka[i % 3][j];
                if constexpr (I8) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const half8_t kf = half ? i8_to_half8(kw[2], kw[3]) : i8_to_half8(kw[0], kw[1]);
                        const int ks = (i >> 1) * 4 + half * 2 + (i & 1);
                        s[j] = mfma32<KVF>(kf, qh[ks], s[j]);
                        if constexpr (F32) s[j] = mfma32<KVF>(kf, ql[ks], s[j]);
                    }
                } else {
                    const frag kf = __builtin_bit_cast(frag, kw);
                    s[j] = mfma32<KVF>(kf, qh[i], s[j]);
                    if constexpr (F32) s[j] = mfma32<KVF>(kf, ql[i], s[j]);
                }
            }
            if constexpr (!MASK) __builtin_amdgcn_sched_barrier(0);  // in this order
        }
        float vexp = 0.f;
        if constexpr (I8) {
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const size_t at = token_of(cur.blk[j], cur.page[j]) + 8 * hk;
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    const half8_t ksc = *(const half8_t*)(a.pool.ks + at + 16 * g);
                    const half8_t vs = *(const half8_t*)(a.pool.vs + at + 16 * g);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        s[j][8 * g + i] *= (float)ksc[i];
                        const float v = (float)vs[i];
                        vsc[j][8 * g + i] = v;
                        top = fmaxf(top, !MASK || t0[j] + 16 * g + 8 * hk + i < max(w_hi + 1, t.pre) ? v : 0.f);
                    }
                }
            }
            top = half_max(top);
            vexp = top > 0x1p-20f ? (float)__builtin_amdgcn_frexp_expf(top) : -20.f;
        }
        // scores to powers of two: exponent = s * c - ref.  A capped score whose block needs no mask goes
        // from the product to the weight in one go further down.
        if constexpr (MODE != 0) if (!direct) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float at = slope * (float)(t0[j] + 8 * hk - pos);
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float x = s[j][i] * qs;
                    if (MODE == 1 || capped) x = a.softcap * tanh_f32<F32>(x * inv_cap);
                    s[j][i] = fmaf(x, PA_LOG2E, fmaf(slope, (float)(16 * (i >> 3) + (i & 7)), at));
                }
            }
        }
        if constexpr (MASK) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t seen = w.skip[j] ? 0u : seen_bits(t0[j] + 8 * hk, a.window ? max(0, pos - a.window + 1) : 0, pos, t.pre, 32);
#pragma unroll
                for (int i = 0; i < 16; i++) s[j][i] = (seen >> (16 * (i >> 3) + (i & 7))) & 1u ? s[j][i] : -INFINITY;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int i = 1; i < 16; i++) mx = fmaxf(mx, s[0][i]);
#pragma unroll
        for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[1][i]);
        mx = half_max(mx);
        mx = direct ? cap2 * tanh_f32<F32>(mx * qs * inv_cap) : mx * c;
        if constexpr (I8) mx += vexp;
        w.mx = mx;
        return true;
    };
    // O's reference follows the maximum
    auto raise = [&](float mx) __attribute__((always_inline)) {
        const float mn = fmaxf(mx_run, mx);
        const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx_run - mn);
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] *= alpha;
        mx_run = mn;
    };
    auto add = [&](const Step& cur, int buf, auto mask, Work& w) __attribute__((always_inline)) {
        constexpr bool MASK = mask.value;
        constexpr bool direct = !MASK && MODE == 1;
        const float c = factor(mask);
        float16_t(&s)[2] = w.s;
        auto& vsc = w.vsc;
        const int t0[2] = {cur.blk[0] * PAGE_BLK, cur.blk[1] * PAGE_BLK};
        const char* vb = pf_lds + buf * (4 * BLK) + 2 * BLK;
        const float ref = (mx_run == -INFINITY ? 0.f : mx_run) - Mat<KVF>::P_BITS;
        if constexpr (direct) {
            const float k2 = 2.f * c * inv_cap;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    if constexpr (F32) s[j][i] = __builtin_amdgcn_exp2f(cap2 * tanh_f32<true>(s[j][i] * qs * inv_cap) - ref);
                    else s[j][i] = __builtin_amdgcn_exp2f(-2.f * cap2 * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[j][i] * k2) + 1.f) + (cap2 - ref));
                }
        } else {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[j][i] = __builtin_amdgcn_exp2f(fmaf(s[j][i], c, -ref));
        }
        auto v_at = [&](int j, int g, int d) __attribute__((always_inline)) { return *(const u32x4_t*)(vb + j * BLK + (v_lane ^ (g * 32)) + d * 2048); };
        // tokens that no row of this wave sees may hold anything, also NaN
        auto keep_of = [&](int j, int g) __attribute__((always_inline)) {
            return keep_words(w.skip[j] ? 0u : seen_bits(t0[j] + 16 * g + 8 * hk, wlow, w_hi, t.pre, 8));
        };
        bool odd = false;
        if constexpr (MASK && !I8) {
            bool mixed = false;  // blocks of which the rows of this wave see different tokens
#pragma unroll
            for (int j = 0; j < 2; j++)
                mixed |= !w.skip[j] && t0[j] + PAGE_BLK > t.pre && (t0[j] + PAGE_BLK - 1 > w_lo || (a.window && t0[j] <= w_hi - a.window));
            if (mixed && w_lo < w_hi) {
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        const u32x4_t keep = keep_of(j, g);
#pragma unroll
                        for (int d = 0; d < DT; d++) top = Odd<KVF>::top(v_at(j, g, d) & keep, top);
                    }
                odd = Odd<KVF>::any(top);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int g = 0; g < 2; g++) {
                frag ph, pl;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float p = s[j][8 * g + i];
                    l += p;
                    if constexpr (I8) {
                        // a token that is not there may have any scale
                        p = MASK && p == 0.f ? 0.f : p * vsc[j][8 * g + i];
                    }
                    ph[i] = (elem)p;
                    if constexpr (F32) pl[i] = (elem)(p - (float)ph[i]);
                }
                u32x4_t keep;
                if constexpr (MASK && !I8) keep = keep_of(j, g);
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    frag va;
                    if constexpr (I8) {
                        const uint2 vw = *(const uint2*)(vb + j * BLK + v_lane + d * 1024 + g * 512);
                        va = i8_to_half8(vw.x, vw.y);
                    } else {
                        u32x4_t vw = v_at(j, g, d);
                        if constexpr (MASK) {
                            vw &= keep;
                            if (__builtin_expect(odd, 0)) {
                                const frag seen = Odd<KVF>::seen(w.skip[j] ? 0u : seen_bits(t0[j] + 16 * g + 8 * hk, a.window ? max(0, pos - a.window + 1) : 0, pos, t.pre, 8));
                                const float16_t c = mfma32<KVF>(Odd<KVF>::marks(vw), seen, float16_t{});
#pragma unroll
                                for (int i = 0; i < 16; i++) o[d][i] += Odd<KVF>::worth(c[i]);
                                vw = Odd<KVF>::finite(vw);
                            }
                        }
                        va = __builtin_bit_cast(frag, vw);
                    }
                    o[d] = mfma32<KVF>(va, ph, o[d]);
                    if constexpr (F32) o[d] = mfma32<KVF>(va, pl, o[d]);
                }
            }
        if constexpr (!MASK && !I8) {
            // V operands are read four products early (left alone, the compiler reads each just before its product)
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int i = 0; i < 4 * DT - 4; i++) {
                __builtin_amdgcn_sched_group_barrier(0x8, F32 ? 2 : 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, F32 ? 8 : 4, 0);
        }
    };

    bool bad = false;
    Step cur{}, nxt{}, far{};
    if (k0 < k1) {
        nxt = settle(look_up(k0));
        far = look_up(k0 + 2);
        pieces(load_of(nxt, 0));
    }
    const int whole_lo = a.window ? t.p_hi - a.window + 1 : 0;  // tokens from here to p_lo are seen by every row
    int k = k0, buf = 0;
    // next step: its data has landed for every wave, and the other stage is free for the one after it
    auto advance = [&]() __attribute__((always_inline)) {
        cur = nxt;
        wait_vmcnt<0>();
        __syncthreads();
        if (k + 2 < k1) {
            nxt = settle(far);
            far = look_up(k + 4);
        }
        return load_of(nxt, buf ^ 1);  // (the last step loads itself again: nobody reads that)
    };
    auto whole = [&](const Step& s) {
        return (k + 1 < k1) & (s.page[0] >= 0) & (s.page[1] >= 0) & (s.blk[1] * PAGE_BLK + PAGE_BLK - 1 <= t.p_lo) &
               (s.blk[0] * PAGE_BLK >= whole_lo);
    };
    for (;;) {
        // Steps that need no mask, while the maximum stays: nothing in this loop touches O but the products, and it
        // keeps its registers (a conditional factor cost 64 copies a step).
        bool landed = false;
        while (whole(nxt)) {
            const Load ld = advance();
            Work w;
            scores(cur, buf, true, &ld, std::false_type{}, w);
            landed = __any(w.mx > mx_run + Mat<KVF>::P_LAG);
            if (landed) break;  // made again below
            add(cur, buf, std::false_type{}, w);
            k += 2;
            buf ^= 1;
        }
        if (!landed) {  // (otherwise the next step's pieces are on their way)
            if (k >= k1) break;
            pieces(advance());
        }
        bad |= cur.page[0] < 0 || cur.page[1] < 0;
        Work w;
        if (scores(cur, buf, k + 1 < k1, nullptr, std::true_type{}, w)) {
            if (__any(w.mx > mx_run + Mat<KVF>::P_LAG)) raise(w.mx);
            add(cur, buf, std::true_type{}, w);
        }
        k += 2;
        buf ^= 1;
    }
    wait_vmcnt<0>();  // nothing is under way into LDS when the workgroup ends
    if (bad && a.bt.status && tid == 0) atomicOr(&a.bt.status[t.b], PAGE_SEQ_BAD_PAGE);
    l = half_sum(l);
    if (r >= rows) return;
    const long long row = t.s.row0 + tok;
    if (splits > 1) {
        const long long slot = row * a.n_heads + h;
        float* po = part_o(a, split, slot) + 4 * hk;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *(float4_t*)(po + 32 * d + 8 * g) = float4_t{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
        if (hk == 0) *part_ml(a, splits, split, slot) = float2_t{mx_run, l};
        return;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    T* out = (T*)a.out + row * a.out_ld + (long long)h * HD + 4 * hk;
    typedef T out4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *(out4*)(out + 32 * d + 8 * g) = out4{(T)(o[d][4 * g] * inv), (T)(o[d][4 * g + 1] * inv), (T)(o[d][4 * g + 2] * inv),
                                                  (T)(o[d][4 * g + 3] * inv)};
}

// ---------------------------------------------------------------------------
// launch plan
// ---------------------------------------------------------------------------
constexpr int PA_CUS = 256;  // compute units of the part

struct Plan {
    bool prompt;
    int nt, tiles, splits, per;  // 16-row column tiles of a workgroup, tiles of a (sequence, kv head), splits, blocks each
};

Plan plan_of(const PagedAttnArgs& a) {
    const int group = a.n_heads / a.pool.n_kv;
    const long long rows = (long long)a.bt.max_rows * group;
    Plan p{};
    // Tiles of 16 or 32 rows stream the cache through the registers, each tile by itself (from the die's cache after the first);
    // tiles of 128 rows share it through LDS and take longer to start.  The former are quicker for one tile of 32 and
    // while there is little to do in all: few tiles, few blocks for them.  Measured, in us (tiles of 16 or 32 / of
    // 128): fp16, head_dim 128, 4 heads a kv head, sequences x rows over tokens: 1 x 256 over 256 12 / 21, 1 x 160 over 2000
    // 26 / 32, over 8000 83 / 51, 8 x 16 over 4096 41 / 41, 8 x 24 62 / 47, 32 x 12 253 / 120, 4 x 128 over 0 14 / 11;
    // head_dim 64, 12 heads: 16 x 64 over 1000 19 / 25, 16 x 128 29 / 30, over 4096 98 / 81; f32
    // over INT8 (whose codes 128-row tiles convert in every wave): 1 x 64 27 / 49, 8 x 40 105 / 143, 8 x 64 over 8000 157 / 189.
    const long long pairs = (long long)a.bt.nseq * a.pool.n_kv;
    const int seen = a.window && !a.prefix ? (int)std::min<long long>(a.bt.max_kv, (long long)a.window + a.bt.max_rows) : a.bt.max_kv;
    const long long f = (a.pool.hd == 64 ? 2 : 1) * (a.pool.fmt == KV_INT8 ? 8 : 1);
    p.prompt = rows > 32 && (rows * pairs > 8192 * f || rows * pairs * ((seen + 31) / 32) > 540000 * f);
    // One 16-row tile a workgroup where that leaves every workgroup a compute unit of its own or wastes less than 32-row tiles,
    // which read the cache half as often (8 rows x 4 heads, 4096 tokens: 1 sequence 13 us and 16, 32 sequences 146 and 91;
    // 33 rows over 1000, 16 x 12 heads of 64: 14.5 and 18.5).
    const long long tiles16 = (rows + 15) / 16;
    p.nt = tiles16 == 1 || tiles16 == 3 || pairs * tiles16 <= (a.pool.hd == 64 && tiles16 > 2 ? 2 : 1) * PA_CUS ? 1 : 2;
    const int tile_rows = p.prompt ? PF_ROWS : 16 * p.nt;
    p.tiles = (int)((rows + tile_rows - 1) / tile_rows);
    // blocks that a tile can visit
    const int all = (a.bt.max_kv + 31) / 32;
    const int span = (tile_rows + group - 1) / group + 1;
    const int n = a.window && !a.prefix ? (int)std::min<long long>(all, ((long long)a.window + span) / 32 + 2) : all;
    const long long base = (long long)a.bt.nseq * a.pool.n_kv * p.tiles;
    const int unit = p.prompt ? 2 : dc_waves(a.pool.fmt);  // blocks of a step (prompt) or of a round of the waves
    if (p.prompt) {
        // Fewer steps for a workgroup against more partial results and a second launch.  Measured at head_dim 128, fp16: 1.5 us
        // a step with one workgroup on a compute unit, 2 us each with two; 3 us to start, 4 us and 3.5 TB/s to join.
        const double step = (0.5 + a.pool.hd / 128.0) * (a.act == ACT_F32 ? 1.6 : 1.0) * (a.pool.fmt == KV_INT8 ? 1.3 : 1.0);
        double best = 0;
        p.splits = 1;
        for (int k = 1; k <= std::min(32, std::max(1, n / 4)); k++) {
            const double per_cu = std::ceil((double)(base * k) / PA_CUS);
            const double steps = std::ceil((n + 1) / 2 / (double)k);
            double us = (3 + steps * step) * (per_cu <= 1 ? 1.0 : per_cu * 0.67);
            if (k > 1) us += 4 + (double)a.bt.rows * a.n_heads * k * (a.pool.hd + 2) * 8 / 3.5e6;
            if (k == 1 || us < 0.95 * best) {
                best = us;
                p.splits = k;
            }
        }
    } else {
        // A block for each wave, and as many workgroups as compute units (twice as many at head_dim 64: 10 x 12 heads over
        // 4096 27 us and 31; at 128 32 x 4 rows over INT8 60 and 51) but not more, so that they end together (20 x 8 kv heads:
        // 160 workgroups 58 us, 320 68).  64 splits at most: a lane each when they are joined.
        p.splits = (int)std::min<long long>(std::min(64, std::max(1, n / unit)), std::max<long long>(1, (a.pool.hd == 64 ? 2 : 1) * PA_CUS / base));
    }
    p.per = (n + p.splits - 1) / p.splits;
    p.per = (p.per + unit - 1) / unit * unit;
    p.splits = std::max(1, (n + p.per - 1) / p.per);
    return p;
}

template <typename T, int KVF, int HD>
int launch_hd(const PagedAttnArgs& a, hipStream_t stream) {
    const Plan p = plan_of(a);
    const int group = a.n_heads / a.pool.n_kv;
    const long long blocks = (long long)a.bt.nseq * a.pool.n_kv * p.tiles * p.splits;
    if (blocks > 0x7fffffffLL / 256) return note_error(hipErrorInvalidConfiguration);  // (the entry refuses such calls)
    const dim3 grid((unsigned)blocks);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(p.prompt ? 256 : dc_waves(KVF) * 64), 0, stream, a, group, p.tiles, p.splits, p.per); };
    if (p.prompt && a.slopes) go(paged_prompt_kernel<T, KVF, HD, 2>);
    else if (p.prompt && a.softcap > 0.f) go(paged_prompt_kernel<T, KVF, HD, 1>);
    else if (p.prompt) go(paged_prompt_kernel<T, KVF, HD, 0>);
    else if (p.nt == 1 && p.tiles == 1) go(paged_decode_kernel<T, KVF, HD, 1, true>);
    else if (p.nt == 1) go(paged_decode_kernel<T, KVF, HD, 1, false>);
    else if (p.tiles == 1) go(paged_decode_kernel<T, KVF, HD, 2, true>);
    else go(paged_decode_kernel<T, KVF, HD, 2, false>);
    if (p.splits > 1) {
        // Measured: 500 rows x 32 heads in 4 splits 8.5 us, 13.5 with a slot a wave; 1 x 32 in 32 splits 4.0 us, 5.6 with a wave a slot
        const long long n = (long long)a.bt.max_rows * a.n_heads;
        auto join = [&](auto kernel, int slots) {  // slots of a workgroup
            hipLaunchKernelGGL(kernel, dim3((unsigned)((n + slots - 1) / slots), a.bt.nseq), dim3(256), 0, stream, a, p.splits);
        };
        if (p.splits <= 512 / HD && n * a.bt.nseq > 4096) join(paged_merge_kernel<T, HD, 4, 1>, 16);
        else if (p.splits > 8 && n * a.bt.nseq <= 1024) join(paged_merge_kernel<T, HD, 1, 4>, 1);
        else join(paged_merge_kernel<T, HD, 1, 1>, 4);
    }
    return note_error(hipGetLastError());
}

template <typename T, int KVF>
int launch_kv(const PagedAttnArgs& a, hipStream_t stream) {
    return a.pool.hd == 128 ? launch_hd<T, KVF, 128>(a, stream) : launch_hd<T, KVF, 64>(a, stream);
}

}  // namespace

long long paged_attention_workspace(const PagedAttnArgs& a) {
    const Plan p = plan_of(a);
    return p.splits > 1 ? (long long)p.splits * a.bt.rows * a.n_heads * (a.pool.hd + 2) * 4 : 0;
}

int launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
    if (a.act == ACT_F32)
        return a.pool.fmt == KV_INT8 ? launch_kv<float, KV_INT8>(a, stream) : launch_kv<float, KV_F16>(a, stream);
    if (a.act == ACT_F16)
        return a.pool.fmt == KV_INT8 ? launch_kv<_Float16, KV_INT8>(a, stream) : launch_kv<_Float16, KV_F16>(a, stream);
    return launch_kv<__bf16, KV_BF16>(a, stream);
}

}  // namespace aarh
