// Tile arithmetic of the attention kernels (attention.hip, attention_bwd.hip): fragments, matrix products, masks and the
// relative-position bias, the same code for f32, bf16 and f16.
//
// One convention carries every kernel.  A score tile is formed so that its CONTRACTED-NEXT dimension lies in the registers of a lane and
// the other one on the lanes: forward and dq hold S^T (lane = query row, registers = keys), dk / dv hold S (lane = key, registers =
// query rows).  Row statistics of the forward are then lane-local, and the tile feeds the next product as its B operand straight from
// registers: the register order of a C tile (quads of four consecutive rows, one quad per lane group) is used as the ORDER OF THE
// CONTRACTION, and the other operand is fetched in the same order -- by transposing LDS reads for 16-bit types, by plain reads for f32.
#pragma once
#include "common.h"
#include "../../include/ekaid_hip.h"

namespace ekaid {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int ATTN_MAX_BUCKETS = EKAID_ATTN_MAX_BUCKETS;
constexpr float NEG_INF = -__builtin_inff(), POS_INF = __builtin_inff();
constexpr float LOG2E = 1.4426950408889634f;

struct AttnArgs {
    ekaid_attn_t d;                   // the caller's descriptor (strides, masks, table, dropout)
    DropSeed seed;
    float inv_keep;
    float sc2;                        // scale * log2(e): the softmax runs on powers of two
    int gp;                           // heads packed into the rows of one workgroup (row r = query r / gp, head r % gp): 1 or H / KV
    int tiles;                        // row tiles (forward, dq) / key tiles (dk, dv)
    int splits;                       // workgroups that share a row tile's keys (forward, dq) / a key tile's rows (dk, dv)
    int dq_parts;                     // row-norm words per head that dq wrote (f16)
    float* po;                        // partial outputs of a split launch [splits][...]
    float* pml;                       // their (max, sum) pairs
    float* delta;                     // [B][H][Lq]
    float* nrm;                       // [B * H][dq_parts]
    float* ptab;                      // [B * H][dq_parts][nb]
    float* pk;                        // partial dk, dv
    float* pv;
};

template <typename T> struct Elem;
template <> struct Elem<float> { static constexpr int epl = 4; };
template <> struct Elem<__bf16> { static constexpr int epl = 8; };
template <> struct Elem<_Float16> { static constexpr int epl = 8; };

// G = edge of a score block (32 or 16): 64 / G lane groups, each lane holds G * G / 64 values in quads
template <int G> struct Blk;
template <> struct Blk<32> { typedef f32x16 acc; static constexpr int ng = 2, nq = 4; };
template <> struct Blk<16> { typedef f32x4 acc; static constexpr int ng = 4, nq = 1; };

template <int G> __device__ __forceinline__ typename Blk<G>::acc zero_acc() {
    typename Blk<G>::acc z;
#pragma unroll
    for (int i = 0; i < 4 * Blk<G>::nq; ++i) z[i] = 0.f;
    return z;
}

// c += a b over one 16-byte fragment per lane: 16 (G = 32) or 32 (G = 16) contracted 16-bit elements, 8 or 16 in f32
template <typename T, int G> __device__ __forceinline__ typename Blk<G>::acc mma(u32x4 a, u32x4 b, typename Blk<G>::acc c) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (G == 32) c = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[e], fb[e], c, 0, 0, 0);
            else c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[e], fb[e], c, 0, 0, 0);
        }
    } else if constexpr (__is_same(T, __bf16)) {
        const bf16x8 x = __builtin_bit_cast(bf16x8, a), y = __builtin_bit_cast(bf16x8, b);
        if constexpr (G == 32) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
        else c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
    } else {
        const f16x8 x = __builtin_bit_cast(f16x8, a), y = __builtin_bit_cast(f16x8, b);
        if constexpr (G == 32) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
        else c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
    }
    return c;
}

// two f32 values rounded to nearest and packed
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
template <typename T> __device__ __forceinline__ float elem(u32x4 v, int e) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(f32x4, v)[e];
    else if constexpr (__is_same(T, __bf16)) return (float)__builtin_bit_cast(bf16x8, v)[e];
    else return (float)__builtin_bit_cast(f16x8, v)[e];
}

// fragment of contracted chunk c taken from score registers (values already final): quads 2c, 2c+1 (16-bit) or quad c (f32)
template <typename T, int G, int NB> __device__ __forceinline__ u32x4 score_frag(const typename Blk<G>::acc (&s)[NB], int c) {
    constexpr int nq = Blk<G>::nq;
    u32x4 f;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = __builtin_bit_cast(uint32_t, (float)s[c / nq][4 * (c % nq) + e]);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int q = 2 * c + h;
            f[2 * h] = pack2<T>(s[q / nq][4 * (q % nq)], s[q / nq][4 * (q % nq) + 1]);
            f[2 * h + 1] = pack2<T>(s[q / nq][4 * (q % nq) + 2], s[q / nq][4 * (q % nq) + 3]);
        }
    }
    return f;
}

// A operand whose rows are the COLUMNS of a row-major LDS tile X[row][ld]: columns m0 .. m0+G, contracted over the tile rows in the
// order of score_frag(c).  16-bit: ds_read_b64_tr_b16 -- the 16 lanes of a group read 4 rows x 16 columns and each receives one column.
template <typename T, int G> __device__ __forceinline__ u32x4 col_frag(const T* X, int ld, int m0, int c, int lane) {
    constexpr int ng = Blk<G>::ng;
    const int g = lane / G;
    u32x4 f;
    if constexpr (sizeof(T) == 4) {
        const float* p = reinterpret_cast<const float*>(X) + (c * 4 * ng + 4 * g) * ld + m0 + (lane % G);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = __builtin_bit_cast(uint32_t, p[e * ld]);
    } else {
        const int col = m0 + (G == 32 ? (lane & 16) : 0) + 4 * (lane & 3);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = (2 * c + h) * 4 * ng + 4 * g + ((lane & 15) >> 2);
            typedef __attribute__((address_space(3))) s16x4* lds_t;
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(X + row * ld + col));
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            const u32x2 w = __builtin_bit_cast(u32x2, v);
            f[2 * h] = w[0];
            f[2 * h + 1] = w[1];
        }
    }
    return f;
}
// A or B operand from a row-major LDS tile: row r0 + lane % G, contracted columns of chunk c
template <typename T, int G> __device__ __forceinline__ u32x4 row_frag(const T* X, int ld, int r0, int c, int lane) {
    constexpr int epl = Elem<T>::epl;
    return *reinterpret_cast<const u32x4*>(X + (r0 + lane % G) * ld + (c * Blk<G>::ng + lane / G) * epl);
}
// the same straight from memory (zero beyond column dh, or when the row does not exist)
template <typename T, int G> __device__ __forceinline__ u32x4 row_frag_global(const T* row, int c, int dh, bool ok, int lane) {
    constexpr int epl = Elem<T>::epl;
    const int col = (c * Blk<G>::ng + lane / G) * epl;
    u32x4 z = {0u, 0u, 0u, 0u};
    if (ok && col < dh) z = *reinterpret_cast<const u32x4*>(row + col);
    return z;
}

// LDS leading dimensions (elements): rows read 16 bytes per lane want an odd number of 16-byte slots; columns read by transposition want
// consecutive rows 64 bytes apart modulo the 256-byte bank round (16-bit) or an offset of 8 floats (f32, two lane groups)
template <typename T, int DH> struct Ld {
    static constexpr int row = DH + 16 / (int)sizeof(T);
    static constexpr int col = sizeof(T) == 4 ? DH + 8 : DH + 32;
};

// rows [r0, r0 + ROWS) of a row-major matrix into registers (zero where the row index reaches `limit`, the key mask is 0 or the column
// is beyond dh), then from registers into an LDS tile.  Masked rows never enter a product: NaN or Inf in them stays there.
template <typename T, int DH, int ROWS, int NT> struct Stage {
    static constexpr int epl = Elem<T>::epl, vpr = DH / epl, n = ROWS * vpr, per = (n + NT - 1) / NT;
    u32x4 r[per];
    __device__ __forceinline__ void load(const T* base, long long stride, int r0, int limit, int dh, const unsigned char* mask, int tid) {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int id = i * NT + tid, row = id / vpr, col = (id % vpr) * epl;
            u32x4 z = {0u, 0u, 0u, 0u};
            const int gr = r0 + row;
            if (id < n && gr < limit && col < dh && (!mask || mask[gr])) z = *reinterpret_cast<const u32x4*>(base + (long long)gr * stride + col);
            r[i] = z;
        }
    }
    __device__ __forceinline__ void store(T* lds, int ld, int tid) const {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int id = i * NT + tid;
            if (id < n) *reinterpret_cast<u32x4*>(lds + (id / vpr) * ld + (id % vpr) * epl) = r[i];
        }
    }
};

__device__ __forceinline__ long long clamp_index(long long v, long long lo, long long hi) { return v < lo ? lo : v > hi ? hi : v; }
__device__ __forceinline__ int key_len(const ekaid_attn_t& d, int b) {
    if (!d.k_len) return d.Lk;
    const long long n = d.k_len64 ? reinterpret_cast<const long long*>(d.k_len)[b] : (long long)reinterpret_cast<const int*>(d.k_len)[b];
    return (int)clamp_index(n, 0, d.Lk);
}
__device__ __forceinline__ int query_pos(const ekaid_attn_t& d, int b) {
    if (!d.q_pos) return 0;
    const long long n = d.q_pos64 ? reinterpret_cast<const long long*>(d.q_pos)[b] : (long long)reinterpret_cast<const int*>(d.q_pos)[b];
    return (int)clamp_index(n, -(1 << 29), 1 << 29);
}

// bucket of the offset key - query: the number of borders at or below the distance, upper half for keys ahead (both directions)
__device__ __forceinline__ int rel_bucket(const ekaid_attn_t& d, int rel) {
    const int dist = d.bidirectional ? (rel < 0 ? -rel : rel) : (rel < 0 ? -rel : 0);
    int b = 0;
    for (int i = 0; i < d.n_border; ++i) b += dist >= d.border[i] ? 1 : 0;
    return b + (d.bidirectional && rel > 0 ? d.n_border + 1 : 0);
}
__device__ __forceinline__ float table_at(const ekaid_attn_t& d, int bucket, int head) {
    const long long i = (long long)bucket * d.H + head;
    if (d.table_dtype == EKAID_F32) return reinterpret_cast<const float*>(d.table)[i];
    if (d.table_dtype == EKAID_BF16) return (float)reinterpret_cast<const __bf16*>(d.table)[i];
    return (float)reinterpret_cast<const _Float16*>(d.table)[i];
}
// bias of `heads` heads by clamped distance, in units of the power-of-two softmax: bias[h][rel + reach], rel in [-reach, reach]
__device__ __forceinline__ void fill_bias(const ekaid_attn_t& d, float* bias, int head0, int heads, int tid, int nt) {
    const int w = 2 * d.reach + 1;
    for (int i = tid; i < heads * w; i += nt) bias[i] = table_at(d, rel_bucket(d, i % w - d.reach), head0 + i / w) * LOG2E;
}

// which workgroup works on what: consecutive work items (tiles of one head, which share their keys) on ONE die -- workgroups are dealt
// to the 8 dies in turn, each die has its own L2
__device__ __forceinline__ int die_order(int bid, int n) {
    const int x = bid & 7, q = n >> 3, r = n & 7;
    return x * q + (x < r ? x : r) + (bid >> 3);
}

template <int G> __device__ __forceinline__ float across_groups_max(float v) {
#pragma unroll
    for (int o = G; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
template <int G> __device__ __forceinline__ float across_groups_sum(float v) {
#pragma unroll
    for (int o = G; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}
template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float e) {
    if constexpr (sizeof(T) == 4) { f32x4 v = {a, b, c, e}; *reinterpret_cast<f32x4*>(p) = v; }
    else {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        u32x2 v = {pack2<T>(a, b), pack2<T>(c, e)};
        *reinterpret_cast<u32x2*>(p) = v;
    }
}
// LDS hand-off between the lanes of one wave
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ float drop_keep(const AttnArgs& a, uint64_t seed, int b, int h, int i, int j) {
    const uint64_t idx = (((uint64_t)b * a.d.H + h) * a.d.Lq + i) * (uint64_t)a.d.Lk + j;
    return dropout_scale(seed, idx, a.d.drop_p, a.inv_keep);
}

// scores of one key tile, s[sub] = K Q^T (raw products) -> masked, biased, in powers of two.  Lane: one query row (position pos, head
// row `bias`), registers: keys j0 + 4 ng quad + 4 g + e.
template <int G, int NB>
__device__ __forceinline__ void finish_scores(const AttnArgs& a, typename Blk<G>::acc (&s)[NB], int j0, int len, int pos, const float* bias,
                                              const unsigned char* km, bool partial, int lane) {
    constexpr int ng = Blk<G>::ng, nq = Blk<G>::nq;
    const int g = lane / G, reach = a.d.reach;
#pragma unroll
    for (int q = 0; q < NB * nq; ++q) {
        const int jq = 4 * ng * q + 4 * g;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = s[q / nq][4 * (q % nq) + e] * a.sc2;
            const int j = j0 + jq + e;
            if (bias) x += bias[min(max(j - pos, -reach), reach) + reach];
            if (partial && !(j < len && (!km || km[jq + e]) && (!a.d.causal || j <= pos))) x = NEG_INF;
            s[q / nq][4 * (q % nq) + e] = x;
        }
    }
}

struct RowWork {                       // one workgroup's share of the forward / dq work list
    int b, head0, kvh, tile, split;
    __device__ __forceinline__ RowWork(const AttnArgs& a) {
        const int nhg = a.d.H / a.gp, w = die_order(blockIdx.x, gridDim.x);
        tile = w % a.tiles;
        if (a.d.causal) tile = a.tiles - 1 - tile;        // the longest rows first
        const int rest = w / a.tiles;
        split = rest % a.splits;
        const int bh = rest / a.splits;
        b = bh / nhg;
        head0 = (bh % nhg) * a.gp;
        kvh = head0 / (a.d.H / a.d.KV);
    }
};

int attn_check(const ekaid_attn_t* a, const char* who);
size_t attn_bwd_workspace(const ekaid_attn_t* a);

}  // namespace ekaid
