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
#include <type_traits>
#include <utility>
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
    int near;                         // key heads next to each other in the work list (divides KV)
    int tiles;                        // row tiles (forward, dq) / key tiles (dk, dv)
    int splits;                       // workgroups that share a row tile's keys (forward, dq) / a key tile's rows (dk, dv)
    int dq_parts;                     // row-norm words per head that dq wrote (f16)
    float* po;                        // partial outputs of a split launch [splits][...]
    float* pml;                       // their (max, sum) pairs
    float* delta;                     // [B][H][Lq]
    float* nrm;                       // [B * H][dq_parts]
    float* vn;                        // [B * KV][v_parts]: largest squared norms of value rows (f16)
    int v_parts;
    int keep_exp;                     // smallest power of two >= inv_keep
    float* eps;                       // [splits][B][H][Lq] shares of delta's correction (split dq with a bias table)
    float* ptab;                      // [B * H][key tiles * splits][nb]
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

// A or B operand straight from memory: this lane's row, contracted chunk c (zero beyond column dh, or when the row does not exist)
template <typename T, int G> __device__ __forceinline__ u32x4 row_frag_global(const T* row, int c, int dh, bool ok, int lane) {
    constexpr int epl = Elem<T>::epl;
    const int col = (c * Blk<G>::ng + lane / G) * epl;
    u32x4 z = {0u, 0u, 0u, 0u};
    if (ok && col < dh) z = *reinterpret_cast<const u32x4*>(row + col);
    return z;
}

// ---- tiles copied to LDS without passing registers
// A tile is ROWS rows x DH elements, rows packed (no padding: a wave writes 1 KB in lane order), the 16-byte slots of a row permuted by an
// exclusive-or with swz(row) so that both kinds of reads spread over the banks: 16 rows at one slot (row fragments), and 4 consecutive
// rows over 64 or 32 bytes (transposing reads), two rows 4 apart over 128 bytes or four over 64 (f32 columns).  16-byte reads go to the banks
// in groups of lanes 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31: with blocks of 16 rows, where lanes 16 on read the next slot, rows whose
// swz() differ by 1 must lie in one group (dk / dv of 128-wide 16-bit heads: 2 extra cycles of every 8 otherwise).  The permutation is
// applied to the global
// address.  Rows that do not exist, are masked or (causal) lie behind the last position of the workgroup, and columns beyond dh, are read
// from a zero vector: NaN or Inf there never arrives.
__device__ __attribute__((aligned(16))) const uint32_t attn_zero16[4] = {0u, 0u, 0u, 0u};
typedef __attribute__((address_space(3))) void* lds_void;
typedef const __attribute__((address_space(1))) void* global_void;

template <typename T, int DH> __device__ __host__ __forceinline__ constexpr int swz(int row) {
    const int b0 = row & 1, b1 = (row >> 1) & 1, b2 = (row >> 2) & 1, b3 = (row >> 3) & 1;
    if constexpr (DH * sizeof(T) == 128) return b1 << 2 | (b2 ^ b3) << 1 | b3;
    else if constexpr (sizeof(T) == 2) return b0 << 2 | b1 << 3 | (b2 ^ b3) << 1 | b3;
    else return b2 << 3 | b3 << 2 | b1 << 1 | b0;
}
template <typename T, int DH, int ROWS, int NW> struct TileCopy {
    static constexpr int epl = Elem<T>::epl, rb = DH * (int)sizeof(T), per = 1024 / rb > 0 ? 1024 / rb : 1, lanes = rb / 16, chunks = ROWS * rb / 1024 / NW;
    static_assert(rb <= 1024 && chunks >= 1 && chunks * NW * 1024 == ROWS * rb, "");
    const char* lane_base;                     // row lane / lanes of the matrix
    long long stride;                          // bytes between rows
    int lrow, p;
    __device__ __forceinline__ void init(const void* base, long long row_elems, int lane) {
        stride = row_elems * (long long)sizeof(T);
        lrow = lane / lanes;
        p = lane % lanes;
        lane_base = (const char*)base + lrow * stride;
    }
    // rows r0 .. r0 + ROWS of the matrix; km: this tile's key mask in LDS, or NULL
    __device__ __forceinline__ void issue(T* lds, int r0, int limit, int dh, const unsigned char* km, int wave) const {
        const bool whole = r0 + ROWS <= limit && dh == DH && !km;
#pragma unroll
        for (int i = 0; i < chunks; ++i) {
            const int cr = (i * NW + wave) * per, row = cr + lrow, s = p ^ swz<T, DH>(row);
            const char* src = lane_base + (long long)(r0 + cr) * stride + s * 16;
            if (!whole) {
                const bool ok = r0 + row < limit && s * epl < dh && (!km || km[row]);
                src = ok ? src : (const char*)attn_zero16;
            }
            __builtin_amdgcn_global_load_lds((global_void)src, (lds_void)(reinterpret_cast<char*>(lds) + (i * NW + wave) * 1024), 16, 0, 0);
        }
    }
};
// every copy of this wave has landed and every LDS read of it has returned; then the workgroup meets
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
}
// Where a lane finds its part of a fragment.  swz() is linear over exclusive-or and tile rows begin at multiples of 16, so an address is
// (lane part ^ constant) + constant: `row` for fragments of rows, `col` for columns read as rows (contracted in the order of score_frag).
// refresh() hides the lane parts from the optimizer: one exclusive-or per read instead of dozens of addresses kept in registers.
template <typename T, int DH, int G> struct TileFrag {
    static constexpr int ng = Blk<G>::ng, rb = DH * (int)sizeof(T);
    int row, col;
    __device__ __forceinline__ explicit TileFrag(int lane) {
        const int g = lane / G, n = lane % G;
        row = n * rb + ((g ^ swz<T, DH>(n)) << 4);
        if constexpr (sizeof(T) == 4) col = 4 * g * rb + (((n >> 2) ^ swz<T, DH>(4 * g)) << 4) + ((n & 3) << 2);
        else {
            const int r = 4 * g + ((lane & 15) >> 2), slot = (G == 32 ? (lane & 16) >> 3 : 0) | ((lane & 3) >> 1);
            col = r * rb + ((slot ^ swz<T, DH>(r)) << 4) + ((lane & 1) << 3);
        }
    }
    __device__ __forceinline__ void refresh() { asm volatile("" : "+v"(row), "+v"(col)); }
    // rows r0 + n (r0 a multiple of 16), contracted chunk c
    __device__ __forceinline__ u32x4 rows(const T* X, int r0, int c) const {
        return *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(X) + ((row ^ (c * ng * 16)) + r0 * rb));
    }
    // columns m0 + n (m0 a multiple of G), contracted over tile rows r0 + the rows of chunk c
    __device__ __forceinline__ u32x4 cols(const T* X, int m0, int r0, int c) const {
        const char* x = reinterpret_cast<const char*>(X);
        u32x4 f;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = c * 4 * ng + e;              // swz of the constant part of the row
                f[e] = *reinterpret_cast<const uint32_t*>(x + ((col ^ (((m0 >> 2) ^ swz<T, DH>(r)) << 4)) + (r0 + r) * rb));
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = (2 * c + h) * 4 * ng;
                typedef __attribute__((address_space(3))) s16x4* tr_ptr;
                typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
                const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(x + ((col ^ (((m0 >> 3) ^ swz<T, DH>(r)) << 4)) + (r0 + r) * rb)));
                const u32x2 w = __builtin_bit_cast(u32x2, v);
                f[2 * h] = w[0];
                f[2 * h + 1] = w[1];
            }
        }
        return f;
    }
};

template <typename F, int... I> __device__ __forceinline__ void for_each_constant(F& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
// for n in 0 .. N - 1: use(n, load(n)) with the fragments of the next `ahead` steps under way: enough matrix cycles (4 x 64 / 32 in f32, 32 / 16
// in 16 bits a fragment) to cover a fragment's LDS latency.  The order is pinned: left alone, the scheduler either waits for every
// fragment right behind its read or fetches dozens early and spills.
template <typename T, int G, int N, typename Load, typename Use> __device__ __forceinline__ void fragment_loop(Load load, Use use) {
    constexpr int want = sizeof(T) == 4 ? 64 / G - 1 : 128 / G, ahead = want < N ? want : N;
    u32x4 buf[ahead];
#pragma unroll
    for (int n = 0; n < ahead; ++n) buf[n] = load(n);
    auto step = [&](auto c) __attribute__((always_inline)) {
        constexpr int n = decltype(c)::value;
        const u32x4 x = buf[n % ahead];
        if constexpr (n + ahead < N) buf[n % ahead] = load(n + ahead);
        use(n, x);
        __builtin_amdgcn_sched_barrier(0);
    };
    for_each_constant(step, std::make_integer_sequence<int, N>{});
}

// The key mask of the tiles ahead: a byte per key, a ring of four tiles in LDS.  Read from memory three tiles ahead, written a tile later,
// needed two tiles later by the copies and three later by the scores: nobody waits for it.
template <int KT> struct MaskRing {
    const unsigned char* mask;
    unsigned char* ring;
    int len, tid, next;
    __device__ __forceinline__ int at(int t) const { const int j = t * KT + tid; return tid < KT && j < len ? mask[j] : 0; }
    // tiles t .. t + 2; the workgroup meets before the first copy
    __device__ __forceinline__ void init(const unsigned char* m, unsigned char* r, int len_, int t, int tid_) {
        mask = m; ring = r; len = len_; tid = tid_; next = 0;
        if (!mask) return;
        for (int k = 0; k < 3; ++k)
            if (tid < KT) ring[((t + k) & 3) * KT + tid] = (unsigned char)at(t + k);
        next = at(t + 3);
        __syncthreads();
    }
    // at tile t, behind the barrier: tile t + 3 into the ring, tile t + 4 under way
    __device__ __forceinline__ void step(int t) {
        if (!mask) return;
        if (tid < KT) ring[((t + 3) & 3) * KT + tid] = (unsigned char)next;
        next = at(t + 4);
    }
    __device__ __forceinline__ const unsigned char* tile(int t) const { return mask ? ring + (t & 3) * KT : nullptr; }
};

constexpr int BIAS_PAD = 128;          // far values beyond the reach on both sides: a block that touches the reach needs no clamp
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
// in units of the power-of-two softmax.  An entry of -6e4 or less closes its distances like -inf: a row that meets nothing else would have
// such a number as its maximum and denominator, where f32 has no room left for the scores and for the logarithm of the sum.
__device__ __forceinline__ float bias_at(const ekaid_attn_t& d, int rel, int head) {
    const float t = table_at(d, rel_bucket(d, rel), head);
    return t <= EKAID_ATTN_CLOSED ? NEG_INF : t * LOG2E;
}
// bias of `heads` heads by distance: bias[h][rel + reach], rel in [-reach, reach]
__device__ __forceinline__ void fill_bias(const ekaid_attn_t& d, float* bias, int head0, int heads, int tid, int nt) {
    const int w = 2 * d.reach + 1;
    for (int i = tid; i < heads * w; i += nt) bias[i] = bias_at(d, i % w - d.reach, head0 + i / w);
}

// the same for one head, padded, and only the distances `lo` .. `hi` a workgroup meets (and the two of everything beyond the reach)
__device__ __forceinline__ void fill_bias_range(const ekaid_attn_t& d, float* bias, int head, int lo, int hi, int tid, int nt) {
    lo = max(lo, -d.reach - BIAS_PAD);
    hi = min(hi, d.reach + BIAS_PAD);
    for (int rel = lo + tid; rel <= hi; rel += nt) bias[rel + d.reach + BIAS_PAD] = bias_at(d, min(max(rel, -d.reach), d.reach), head);
    if (tid < 2) bias[BIAS_PAD + tid * 2 * d.reach] = bias_at(d, tid ? d.reach : -d.reach, head);
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
// the forward's: 1 or 0 -- the factor of what is kept joins the division by the sum, so that f16 holds the probabilities whatever it is
__device__ __forceinline__ float drop_kept(const AttnArgs& a, uint64_t seed, int b, int h, int i, int j) {
    const uint64_t idx = (((uint64_t)b * a.d.H + h) * a.d.Lq + i) * (uint64_t)a.d.Lk + j;
    return dropout_scale(seed, idx, a.d.drop_p, 1.f);
}
__device__ __forceinline__ float drop_keep(const AttnArgs& a, uint64_t seed, int b, int h, int i, int j) {
    const uint64_t idx = (((uint64_t)b * a.d.H + h) * a.d.Lq + i) * (uint64_t)a.d.Lk + j;
    return dropout_scale(seed, idx, a.d.drop_p, a.inv_keep);
}

// How the raw products of a unit become exponents: exponent = score * mult + add.  Where nothing is masked and the bias is one value (none,
// or all distances beyond the reach) mult / add are that and the scores stay as they are; otherwise they are finished in place (mult 1).
struct Affine { float mult, add; };

// one unit of NB blocks in the S^T orientation (lane: query row at `pos`; registers: keys j0 + 4 ng quad + 4 g + e).  `pmin`, `pmax`:
// positions of this wave's rows; `bias`: padded table of the head (NULL: none); `km`: key mask of the unit (NULL: none)
template <int G, int NB>
__device__ __forceinline__ Affine scores_by_row(const AttnArgs& a, typename Blk<G>::acc (&s)[NB], int j0, int len, int pos, int pmin, int pmax, const float* bias,
                                                const unsigned char* km, int lane) {
    constexpr int ng = Blk<G>::ng, nq = Blk<G>::nq;
    const int g = lane / G, reach = a.d.reach, jn = j0 + NB * G;
    const bool masked = km || jn > len || (a.d.causal && jn - 1 > pmin);
    Affine f = {a.sc2, 0.f};
    bool near = false;
    if (bias) {
        if (jn - 1 - pmin <= -reach) f.add = bias[BIAS_PAD];
        else if (j0 - pmax >= reach) f.add = bias[2 * reach + BIAS_PAD];
        else near = true;
    }
    if (!masked && !near && a.sc2 >= 0.f) return f;
    const float* b = near ? bias + (j0 + 4 * g - pos + reach + BIAS_PAD) : nullptr;
#pragma unroll
    for (int q = 0; q < NB * nq; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = 4 * ng * q + e;
            float x = s[q / nq][4 * (q % nq) + e] * f.mult + f.add;
            if (near) x += b[k];
            s[q / nq][4 * (q % nq) + e] = x;
        }
    if (masked) {
        const int last = a.d.causal ? min(len - 1, pos) : len - 1;        // of this row
#pragma unroll
        for (int q = 0; q < NB * nq; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = s[q / nq][4 * (q % nq) + e];
                s[q / nq][4 * (q % nq) + e] = j0 + 4 * g + 4 * ng * q + e <= last ? x : NEG_INF;
            }
        if (km) {
#pragma unroll
            for (int q = 0; q < NB * nq; ++q) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(km + 4 * ng * q + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = s[q / nq][4 * (q % nq) + e];
                    s[q / nq][4 * (q % nq) + e] = (w >> (8 * e)) & 255u ? x : NEG_INF;
                }
            }
        }
    }
    return Affine{1.f, 0.f};
}

// one workgroup's share of the forward / dq work list.  Order: tile, split, heads that share keys, `near` key heads, sample, the other key
// heads -- what shares keys is together on a die, and every die sees many samples (dealt sample by sample, the die of the longest one
// finishes last: 8 ragged samples in training 103 -> 89 us).  near = 4 for few query rows over up to 512 states, where neighbouring heads share
// pages (64 x 4 heads over 104 f32 states held in the caches: 16 us, 27 with near = 1), else 1 (32 x 16 heads over a cache of 4096: 83 us,
// 94 with near = 4).  Both sides of the border, near = 4 / 1, us, states out of the caches: 64 x 4 heads of 256 f32 over 256 states 33.8 / 36.4,
// 512 58.5 / 60.1, 1024 105.2 / 104.4, 2048 192 / 183; 64 x 16 heads of 64 bf16 over 512 31.9 / 32.9, 1024 59.6 / 57.4, 2048 113 / 100.
struct RowWork {
    int b, head0, kvh, tile, split;
    __device__ __forceinline__ RowWork(const AttnArgs& a) {
        const int w = die_order(blockIdx.x, gridDim.x), group = a.d.H / a.d.KV, shares = group / a.gp;
        tile = w % a.tiles;
        if (a.d.causal) tile = a.tiles - 1 - tile;        // the longest rows first
        int rest = w / a.tiles;
        split = rest % a.splits;
        rest /= a.splits;
        const int share = rest % shares;
        rest /= shares;
        const int lo = rest % a.near;
        rest /= a.near;
        b = rest % a.d.B;
        kvh = rest / a.d.B * a.near + lo;
        head0 = kvh * group + share * a.gp;
    }
};

int attn_check(const ekaid_attn_t* a, const char* who);
int attn_lds_limit(const void* fn, int bytes);      // once per kernel and device: the dynamic LDS it may be launched with
int waves_for_rows(int R, bool wide);
// keys (or rows) a tile of the copying kernels: 16 KB an operand, twice two of them leave room for two workgroups a compute unit
constexpr int attn_kt(int esize, int dh, int g) { return esize == 4 && dh > 128 ? 16 : g == 16 || dh > 128 || (esize == 4 && dh > 64) ? 32 : 64; }
size_t attn_bwd_workspace(const ekaid_attn_t* a);

}  // namespace ekaid
