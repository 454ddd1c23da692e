// Vocabulary loss of a linear layer without its logits, and its gradient (include/ekaid_hip.h: ekaid_linear_loss_t).
//
// 16-bit types: the rows that count (mask != 0) are listed once; products run on tiles of 256 x 256 x 64 (128 x 128 x 64 where
// there are fewer than 128 of them), operands copied to LDS without passing registers, one tile ahead of the matrix instructions.
//   forward   z^T = W x^T per tile -> per-row maximum and sum of the tile's words; a second small kernel joins the tiles
//   backward  per piece of the vocabulary: z again -> dz = (softmax - onehot) mask, rounded to the type, and the bias partials;
//             dW = dz^T x;  dx partials += dz W.   Three products where the formula has three, one more than if logits were kept: at width D
//             forming z again costs 2 D flops a logit, keeping it in f32 8 bytes of traffic -- at 1120 TF and 4.74 TB/s as long from a width
//             of some 950 on, beyond it forming it again is the price of holding no logits (at 2048 2.6 ms of 11.9 below, against 1.2).
// Bound by the matrix instructions and the barrier of each 64-deep tile: 11008 counting rows x 2048 x 65536 bf16: statistics 2.64 ms (1120 TF),
// dz 3.14 (940, it writes 1.4 GB of logit gradients), dW 2.71 (1090), dx 3.49 (850: 688 workgroups, 344 tiles x 2 shares, are 2.7 rounds of 256,
// and f32 partials are read and written once a piece).
// Memory beside the operands: 16-bit dz of a piece of the vocabulary, up to 512 MB (f32: 10 bytes a logit, as five 16-bit planes), up to 16
// f32 partials of dx within 512 MB, and of dW where its tiles are few.
// f32: the same kernels on 16-bit terms of the operands; few words: ll_narrow_*; other arithmetics and small products: passes around
// ekaid_gemm_f32.
#include "common.h"
#include "../../include/ekaid_hip.h"
#include <algorithm>
#include <type_traits>

namespace ekaid {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* global_ptr;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float NEG_INF = -__builtin_inff();
constexpr int BK = 64;
__device__ __attribute__((aligned(16))) const uint32_t zero16[4] = {0u, 0u, 0u, 0u};

// ---- per-call state: [meta: count | sum mask | max |mask| ...][lse2 N][target logit N][nll N][idx N][pos N]
struct State {
    int* count;
    float* sums;         // [0] sum of the mask, [1] max |mask|, [2] largest scale of the weight's rows (f32 terms)
    float* lse;          // log2 denominators, by compact row (16-bit) or by row (f32)
    float* tz;           // target logit in powers of two
    float* nll;          // mask (lse - z_target), by compact row (f32 through ekaid_gemm_f32: by row)
    int* idx;            // compact row -> row
    int* pos;            // row -> compact row, or -1
};
State state_of(void* p, long long n) {
    State s;
    char* c = (char*)p;
    s.count = (int*)c;
    s.sums = (float*)(c + 64);
    s.lse = (float*)(c + 256);
    s.tz = s.lse + n;
    s.nll = s.tz + n;
    s.idx = (int*)(s.nll + n);
    s.pos = s.idx + n;
    return s;
}

// the rows that count, in order; sum and largest magnitude of the mask (thread t: rows t, t + 1024, ...: a fixed order).  One workgroup,
// 16 x 1024 rows at a time: loads together, then one prefix sum over the 256 wave counts.
__global__ __launch_bounds__(1024) void ll_rows_kernel(const float* mask, long long ld, int B, int T, State st) {
    constexpr int U = 16;
    const int n = B * T, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    __shared__ int cnt[U * 16 + 1];
    __shared__ float ssum[1024], smax[16];
    int base = 0;
    float s = 0.f, mx = 0.f;
    for (int r0 = 0; r0 < n; r0 += U * 1024) {
        float m[U];
        unsigned long long on[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int r = r0 + 1024 * k + t;
            m[k] = r < n ? mask[(long long)(r / T) * ld + r % T] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            s += m[k];
            mx = fmaxf(mx, fabsf(m[k]));
            on[k] = __ballot(m[k] != 0.f);
            if (lane == 0) cnt[k * 16 + wave] = __popcll(on[k]);
        }
        __syncthreads();
        if (wave == 0) {                                       // exclusive prefix sums of 256 counts, four a lane
            int c[4], sum = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                c[k] = sum;
                sum += cnt[4 * lane + k];
            }
            int incl = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(incl, o, 64);
                if (lane >= o) incl += v;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) cnt[4 * lane + k] = incl - sum + c[k];
            if (lane == 63) cnt[U * 16] = incl;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int r = r0 + 1024 * k + t;
            if (r >= n) continue;
            const int p = base + cnt[k * 16 + wave] + __popcll(on[k] & ((1ull << lane) - 1));
            const bool mine = m[k] != 0.f;
            if (mine) {
                st.idx[p] = r;
                st.tz[p] = __builtin_nanf("");                 // stays NaN when the target is no word of the vocabulary
            }
            st.pos[r] = mine ? p : -1;
        }
        base += cnt[U * 16];
        __syncthreads();
    }
    ssum[t] = s;
    mx = wave_max(mx);
    if (lane == 0) smax[wave] = mx;
    __syncthreads();
    for (int w = 512; w > 0; w >>= 1) {
        if (t < w) ssum[t] += ssum[t + w];
        __syncthreads();
    }
    if (t == 0) {
        float m = smax[0];
        for (int w = 1; w < 16; ++w) m = fmaxf(m, smax[w]);
        st.count[0] = base;
        st.sums[0] = ssum[0];
        st.sums[1] = m;
    }
}

// ---- tile products of 16-bit operands
template <typename T> __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// One operand tile: R rows (or columns) x 64 contracted elements, 1 KB per wave and instruction straight into LDS.
//   contracted index contiguous (COL = false): LDS [R][64], the 16-byte slots of row r permuted by ^ (r / 2 & 7): 16 rows at one slot fill 64 banks;
//   contracted index strided   (COL = true):  LDS [64][R], the 64-byte groups of row k permuted by ^ (k & 3)
// -- so that fragment reads meet few bank conflicts; the permutation is applied to the GLOBAL address, LDS is written in lane order.
template <int R, bool COL, int NW> struct Operand {
    static constexpr int chunks = R / (8 * NW);
    const char* p[chunks];
    int k0[chunks];                       // first contracted element of this lane's vector (COL: its row), or a large value: read zeros
    long long step;                       // bytes per 64 contracted elements
    long long plane;                      // bytes between the 16-bit planes of an f32 operand
    __device__ __forceinline__ void issue(char* lds, int kt, int pl, int K, int wave) const {
#pragma unroll
        for (int i = 0; i < chunks; ++i) {
            const char* src = kt * BK + k0[i] < K ? p[i] + kt * step + pl * plane : (const char*)zero16;
            __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)(lds + (i * NW + wave) * 1024), 16, 0, 0);
        }
    }
    // row(r): address of row r's first element (any valid address for rows that do not exist)
    template <typename F> __device__ __forceinline__ void init_rows(F row, int wave, int lane) {
        static_assert(!COL, "");
        step = BK * 2;
#pragma unroll
        for (int i = 0; i < chunks; ++i) {
            const int r = (i * NW + wave) * 8 + (lane >> 3), s = (lane & 7) ^ ((r >> 1) & 7);
            p[i] = (const char*)row(r) + s * 16;
            k0[i] = s * 8;
        }
    }
    // element (k, c) at base + k * ld + c; columns from `cols` on read as zero
    __device__ __forceinline__ void init_cols(const void* base, long long ld, int c0, int cols, int wave, int lane) {
        static_assert(COL, "");
        step = ld * BK * 2;
        constexpr int per = R / 8;        // vectors per contracted row
#pragma unroll
        for (int i = 0; i < chunks; ++i) {
            const int k = (i * NW + wave) * (64 / per) + lane / per, s = (lane % per) ^ ((k & 3) << 2), c = c0 + s * 8;
            p[i] = (const char*)base + (k * ld + c) * 2;
            k0[i] = c < cols ? k : 1 << 30;
        }
    }
};
template <int R, bool COL> __device__ __forceinline__ u32x4 operand_frag(const char* lds, int r0, int c, int lane) {
    const int g = lane >> 5;
    if constexpr (!COL) {
        const int r = r0 + (lane & 31);
        return *reinterpret_cast<const u32x4*>(lds + r * 128 + (((c * 2 + g) ^ ((r >> 1) & 7)) << 4));
    } else {
        u32x4 f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = c * 16 + 8 * g + 4 * h + ((lane & 15) >> 2), col = r0 + (lane & 16) + 4 * (lane & 3);
            typedef __attribute__((address_space(3))) s16x4* tr_ptr;
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(lds + k * (R * 2) + (((col >> 3) ^ ((k & 3) << 2)) << 4) + ((col & 7) << 1)));
            const u32x2 w = __builtin_bit_cast(u32x2, v);
            f[2 * h] = w[0];
            f[2 * h + 1] = w[1];
        }
        return f;
    }
}

// f32 operands come as planes of 16-bit terms; their product is the sum of plane products (largest last):
//   3 pairs: two f16 terms an operand (rows scaled by powers of two: 22 significant bits), h h + h l + l h
//   6 pairs: three bf16 terms (exact), the six products above 2^-24
template <int PAIRS> __device__ __forceinline__ int pair_a(int i) { return PAIRS == 1 ? 0 : PAIRS == 3 ? (i == 0) : (0x201100 >> (4 * (5 - i))) & 15; }
template <int PAIRS> __device__ __forceinline__ int pair_b(int i) { return PAIRS == 1 ? 0 : PAIRS == 3 ? (i == 1) : (0x021010 >> (4 * (5 - i))) & 15; }

// acc[mi][ni] += sum over k in [64 kt0, 64 kt1) of A(m, k) B(n, k), for every pair of planes; BM x BN per workgroup, WM x WN per wave.  Two LDS buffers: the copies
// of tile t + 1 are under way while tile t is multiplied; ONE barrier a tile, behind a wait for this wave's copies and LDS reads.
// TURN: the pairs in the order of the product with A and B exchanged, so that both give the same sums.
template <typename T, int BM, int BN, int WM, int WN, bool ACOL, bool BCOL, int PAIRS, bool TURN = false> struct TileProduct {
    static constexpr int NWN = BN / WN, NW = (BM / WM) * NWN, NT = 64 * NW, MI = WM / 32, NI = WN / 32, STAGES = BM == 128 ? 4 : 2;
    typedef Operand<BM, ACOL, NW> A;
    typedef Operand<BN, BCOL, NW> B;
    static __device__ __forceinline__ void step(f32x16 (&acc)[MI][NI], const char* a, const char* b, int wave, int lane) {
        const int m0 = (wave / NWN) * WM, n0 = (wave % NWN) * WN;
#pragma unroll
        for (int c = 0; c < BK / 16; ++c) {
            u32x4 fa[MI], fb[NI];
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[i] = operand_frag<BM, ACOL>(a, m0 + 32 * i, c, lane);
#pragma unroll
            for (int j = 0; j < NI; ++j) fb[j] = operand_frag<BN, BCOL>(b, n0 + 32 * j, c, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = mma32<T>(fa[i], fb[j], acc[i][j]);
        }
    }
    // how many of this wave's copies may still be under way when `newer` tiles behind the one wanted have been asked for
    static __device__ __forceinline__ void arrive(int newer) {
        constexpr int per = A::chunks + B::chunks;            // copies a tile
        static_assert(per == 8, "");
        if (newer >= 2) __builtin_amdgcn_s_waitcnt(0x4070);  // vmcnt 16, lgkmcnt 0
        else if (newer == 1) __builtin_amdgcn_s_waitcnt(0x0078);
        else __builtin_amdgcn_s_waitcnt(0x0070);
        __builtin_amdgcn_s_barrier();
    }
    // K: contracted elements in all (vectors beyond read as zero).  Two buffers where a tile's products (256 x 256: 2 waves a SIMD x 1024
    // matrix cycles) cover the latency of the next tile's copies, four where they do not (128 x 128: 512 cycles) and the grid is small
    // anyway; one barrier a tile: behind it the wanted tile is complete and the buffer of the tile before is free.
    static __device__ __forceinline__ void run(f32x16 (&acc)[MI][NI], const A& oa, const B& ob, int kt0, int kt1, int K, char* a0, char* a1, char* a2, char* a3, char* b0,
                                               char* b1, char* b2, char* b3, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
        if (kt0 < kt1) {
            int kt = kt0, pair = 0;                         // of the tile copied next
            auto copy = [&](char* la, char* lb) __attribute__((always_inline)) {
                oa.issue(la, kt, TURN ? pair_b<PAIRS>(pair) : pair_a<PAIRS>(pair), K, wave);
                ob.issue(lb, kt, TURN ? pair_a<PAIRS>(pair) : pair_b<PAIRS>(pair), K, wave);
                if (++kt == kt1) { kt = kt0; ++pair; }
            };
            const int total = PAIRS * (kt1 - kt0);
            copy(a0, b0);
            if constexpr (STAGES == 2) {
                for (int t = 0; t < total; t += 2) {
                    arrive(0);
                    if (t + 1 < total) copy(a1, b1);
                    step(acc, a0, b0, wave, lane);
                    if (t + 1 < total) {
                        arrive(0);
                        if (t + 2 < total) copy(a0, b0);
                        step(acc, a1, b1, wave, lane);
                    }
                }
            } else {
                if (total > 1) copy(a1, b1);
                if (total > 2) copy(a2, b2);
                for (int t = 0; t < total; t += 4) {
                    arrive(total - 1 - t);
                    if (t + 3 < total) copy(a3, b3);
                    step(acc, a0, b0, wave, lane);
                    if (t + 1 >= total) break;
                    arrive(total - 2 - t);
                    if (t + 4 < total) copy(a0, b0);
                    step(acc, a1, b1, wave, lane);
                    if (t + 2 >= total) break;
                    arrive(total - 3 - t);
                    if (t + 5 < total) copy(a1, b1);
                    step(acc, a2, b2, wave, lane);
                    if (t + 3 >= total) break;
                    arrive(total - 4 - t);
                    if (t + 6 < total) copy(a2, b2);
                    step(acc, a3, b3, wave, lane);
                }
            }
        }
        arrive(0);                                          // the LDS is free for the epilogue
    }
};
// (the copies' buffers are arrays of their own, so that the compiler knows which reads a copy under way concerns)
#define LL_LDS(BM, BN)                                                                                                                                       \
    __shared__ __attribute__((aligned(16))) char la0[BM * BK * 2], la1[BM * BK * 2], lb0[BN * BK * 2], lb1[BN * BK * 2], la2[BM == 128 ? BM * BK * 2 : 16],   \
        la3[BM == 128 ? BM * BK * 2 : 16], lb2[BM == 128 ? BN * BK * 2 : 16], lb3[BM == 128 ? BN * BK * 2 : 16]
#define LL_BUFFERS la0, la1, la2, la3, lb0, lb1, lb2, lb3

// workgroups that share an output tile's contraction: the smallest number that fills the chip's rounds of 256 well, pieces of >= 8 tiles
__host__ __device__ inline int ll_splits(int tiles, int ksteps, int most) {
    int best = 1;
    float filled = 0.f;                                       // (each share writes its own f32 partial tile: no more than needed)
    for (int s = 1; s <= most && (s == 1 || ksteps / s >= 8); ++s) {
        const int wg = tiles * s, rounds = (wg + 255) / 256;
        const float f = rounds ? wg / (256.f * rounds) : 1.f;
        if (filled < 0.85f && f > filled + 0.05f) { filled = f; best = s; }
    }
    return best;
}

struct LossArgs {
    ekaid_linear_loss_t d;
    State st;
    long long nr;             // rows of the compact buffers (multiple of 256)
    int row_tiles;            // upper bound of row tiles (grid)
    int v0, vp;               // first word and words of this piece; ldz = leading dimension of dz
    int ldz;
    float2* part;             // [word tiles][nr] per-row (max, sum) of a tile
    unsigned short* dz;       // [nr][ldz]
    const unsigned short* xc; // [nr][D] the rows that count, zeros behind (f32: [nr][2][D] f16 terms)
    const unsigned short* xb; // f32: [nr][3][D] bf16 terms of the rows that count
    const unsigned short* wp; // the weight (f32: [V][2][D] f16 terms)
    const float* sx;          // f32: powers of two that take the scale of a row of x / of the weight out again
    const float* sw;
    float* up;                // f32: per row, the power of two its dz terms are stored without
    unsigned short* dzb;      // f32: [nr][3][ldz] bf16 terms of dz (dz: [nr][2][ldz] f16 terms of dz sw, for dx)
    float* pdb;               // [row tiles][ldz] bias partials
    float* pdx;               // [splits][nr][D]
    float* pdw;               // [splits][ldz][D] (splits > 1)
    int splits;               // dW: workgroups that share a tile; dx: the most that may
    int* dx_shares;           // the number dx took
    int first_vp;             // words of the first piece (every piece is split like it)
    int first;                // first piece: dx partials are written, later ones added
};

// workgroup -> (row tile, word tile): blocks of 8 word tiles x all row tiles, so that what runs together shares its operands
__device__ __forceinline__ bool ll_tile(int n_row, int n_word, int& rt, int& wt) {
    const int total = n_row * n_word, bid = blockIdx.x;
    if (bid >= total) return false;
    const int x = bid & 7, q = total >> 3, r = total & 7, id = x * q + min(x, r) + (bid >> 3);       // consecutive work on one die
    const int span = 8 * n_row, grp = id / span, left = min(8, n_word - grp * 8), in = id - grp * span;
    wt = grp * 8 + in % left;
    rt = in / left;
    return true;
}

__device__ __forceinline__ float to_f32(const void* p, long long i, int dtype) {
    if (dtype == EKAID_BF16) return (float)reinterpret_cast<const __bf16*>(p)[i];
    if (dtype == EKAID_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
    return reinterpret_cast<const float*>(p)[i];
}

// forward: lanes = rows, registers = words (m), so a row's maximum and sum over the tile are lane-local but for one exchange
// (T: float means f16 terms of f32 operands)
template <typename T> struct Term { typedef T type; static constexpr int planes = 1, pairs = 1; };
template <> struct Term<float> { typedef _Float16 type; static constexpr int planes = 2, pairs = 3; };

template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void ll_stats_kernel(const LossArgs a) {
    typedef TileProduct<typename Term<T>::type, BM, BN, WM, WN, false, false, Term<T>::pairs> P;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int NP = Term<T>::planes;
    LL_LDS(BM, BN);
    const int count = a.st.count[0], tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5;
    int rt, wt;
    if (!ll_tile((count + BN - 1) / BN, (a.d.V + BM - 1) / BM, rt, wt)) return;
    const int w0 = wt * BM, n0 = rt * BN;
    typename P::A oa;
    typename P::B ob;
    oa.init_rows([&](int r) { return (const char*)a.wp + (long long)min(w0 + r, a.d.V - 1) * NP * a.d.D * 2; }, wave, lane);
    ob.init_rows([&](int r) {
        const int n = min(n0 + r, count - 1);
        return F32 ? (const char*)a.xc + (long long)n * NP * a.d.D * 2 : (const char*)a.d.x + a.st.idx[n] * a.d.ldx * 2;
    }, wave, lane);
    oa.plane = ob.plane = (long long)a.d.D * 2;
    f32x16 acc[P::MI][P::NI];
    P::run(acc, oa, ob, 0, (a.d.D + BK - 1) / BK, a.d.D, LL_BUFFERS, wave, lane);
    float* bias = reinterpret_cast<float*>(la0);               // [BM], -inf behind the vocabulary
    float* scale = bias + BM;                                  // [BM] f32: of the word's terms, times log2 e
    float2* red = reinterpret_cast<float2*>(la1);              // [BM / WM][BN]
    for (int i = tid; i < BM; i += P::NT) {
        bias[i] = w0 + i < a.d.V ? (a.d.bias ? to_f32(a.d.bias, w0 + i, a.d.dtype) * LOG2E : 0.f) : NEG_INF;
        if (F32) scale[i] = a.sw[min(w0 + i, a.d.V - 1)] * LOG2E;
    }
    __syncthreads();
    const int wm = wave / P::NWN, wn = wave % P::NWN;
#pragma unroll
    for (int j = 0; j < P::NI; ++j) {
        const int nl = wn * WN + 32 * j + (lane & 31), n = n0 + nl;
        const bool ok = n < count;
        const int row = ok ? a.st.idx[n] : 0;
        const long long tg = ok ? a.d.target[(row / a.d.T) * a.d.ld_target + row % a.d.T] : -1;
        const int tl = tg >= w0 && tg < w0 + BM && tg < a.d.V ? (int)(tg - w0) : -1;
        const float sx = F32 ? a.sx[min(n, count - 1)] : 1.f;
        float mx = NEG_INF, tz = 0.f;
        bool mine = false;
#pragma unroll
        for (int i = 0; i < P::MI; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int ml = wm * WM + 32 * i + 8 * q + 4 * g;
                const f32x4 b4 = *reinterpret_cast<const f32x4*>(bias + ml);
                f32x4 s4 = {LOG2E, LOG2E, LOG2E, LOG2E};
                if (F32) s4 = *reinterpret_cast<const f32x4*>(scale + ml) * sx;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float z = fmaf(acc[i][j][4 * q + e], s4[e], b4[e]);
                    acc[i][j][4 * q + e] = z;
                    mx = fmaxf(mx, z);
                    tz = ml + e == tl ? z : tz;
                    mine |= ml + e == tl;
                }
            }
        if (mine) a.st.tz[n] = tz;
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float base = mx == NEG_INF ? 0.f : mx;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < P::MI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) s += __builtin_amdgcn_exp2f(acc[i][j][r] - base);
        s += __shfl_xor(s, 32, 64);
        if (g == 0) red[wm * BN + nl] = make_float2(mx, s);
    }
    __syncthreads();
    for (int nl = tid; nl < BN; nl += P::NT) {
        float m = NEG_INF, s = 0.f;
#pragma unroll
        for (int w = 0; w < BM / WM; ++w) m = fmaxf(m, red[w * BN + nl].x);
        const float base = m == NEG_INF ? 0.f : m;
#pragma unroll
        for (int w = 0; w < BM / WM; ++w) s += red[w * BN + nl].y * __builtin_amdgcn_exp2f(red[w * BN + nl].x - base);
        if (n0 + nl < count) a.part[(long long)wt * a.nr + n0 + nl] = make_float2(m, s);
    }
}

// lse of a row from its tiles: 64 rows x 16 strands of tiles a workgroup
__global__ __launch_bounds__(1024) void ll_lse_kernel(const LossArgs a, int tiles) {
    __shared__ float sm[16][64], sl[16][64];
    const int r = threadIdx.x & 63, k = threadIdx.x >> 6;
    const long long n = (long long)blockIdx.x * 64 + r;
    const bool ok = n < a.st.count[0];
    float m = NEG_INF, l = 0.f;
    if (ok)
        for (int t = k; t < tiles; t += 16) {
            const float2 p = a.part[t * a.nr + n];
            const float mm = fmaxf(m, p.x), base = mm == NEG_INF ? 0.f : mm;
            l = l * __builtin_amdgcn_exp2f(m - base) + p.y * __builtin_amdgcn_exp2f(p.x - base);
            m = mm;
        }
    sm[k][r] = m;
    sl[k][r] = l;
    __syncthreads();
    if (k || !ok) return;
    for (int i = 1; i < 16; ++i) m = fmaxf(m, sm[i][r]);
    const float base = m == NEG_INF ? 0.f : m;
    l = 0.f;
    for (int i = 0; i < 16; ++i) l += sl[i][r] * __builtin_amdgcn_exp2f(sm[i][r] - base);
    const float lse = m + __builtin_amdgcn_logf(l);
    const int row = a.st.idx[n];
    a.st.lse[n] = lse;
    a.st.nll[n] = (lse - a.st.tz[n]) * LN2 * a.d.mask[(row / a.d.T) * a.d.ld_mask + row % a.d.T];
}

// loss = sum nll / denom, in double and a fixed order
__global__ __launch_bounds__(1024) void ll_loss_kernel(const ekaid_linear_loss_t d, State st, int by_row) {
    __shared__ double s[1024];
    const int count = by_row ? d.B * d.T : st.count[0];
    double x = 0.0;
    for (int n0 = 0; n0 < count; n0 += 8192) {                   // eight loads under way
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = n0 + 1024 * k + (int)threadIdx.x < count ? st.nll[n0 + 1024 * k + threadIdx.x] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) x += (double)v[k];
    }
    s[threadIdx.x] = x;
    __syncthreads();
    for (int w = 512; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) s[threadIdx.x] += s[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) d.loss[0] = (float)(s[0] / (double)(d.denom ? d.denom[0] : st.sums[0]));
}

// compact copy of the rows that count; zero rows up to the next multiple of 64
__global__ __launch_bounds__(256) void ll_gather_kernel(const LossArgs a, unsigned short* xc) {
    const int vec = a.d.D / 8, count = a.st.count[0];
    const long long n = (long long)((count + 255) & ~255) * vec;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256ll * gridDim.x) {
        const int r = (int)(i / vec), c = (int)(i % vec) * 8;
        u32x4 v = {0u, 0u, 0u, 0u};
        if (r < count) v = *reinterpret_cast<const u32x4*>((const unsigned short*)a.d.x + a.st.idx[r] * a.d.ldx + c);
        *reinterpret_cast<u32x4*>(xc + (long long)r * a.d.D + c) = v;
    }
}

template <typename T> __device__ __forceinline__ unsigned short to_bits(float v) { return __builtin_bit_cast(unsigned short, (T)v); }
// (softmax - onehot) mask / max |mask| lies in [-1, 1]; f16 takes it times 2^14, so that probabilities down to 2^-38 keep a value
template <typename T> struct DzScale { static constexpr float up = __is_same(T, _Float16) ? 16384.f : 1.f; };

// output tile through LDS: lanes hold columns, registers rows; bits(value) is what is stored, written as whole 16-byte vectors
template <int BM, int BN, int WM, int WN, int MI, int NI, int NT, typename Bits>
__device__ __forceinline__ void store_tile(const f32x16 (&acc)[MI][NI], Bits bits, unsigned short* out, long long ld, int rows, int cols, char* l0, char* l1, char* l2,
                                           char* l3, int tid, int wave, int lane) {
    constexpr int NWN = BN / WN, Q = BM / 4, HALF = MI / 2;    // a quarter of the rows in each of the four operand buffers: two a wave
    static_assert(Q * BN <= BM * BK && WM == 2 * Q && HALF * 32 == Q, "");
    const int wm = wave / NWN, wn = wave % NWN, g = lane >> 5;
    const int at = 4 * g * BN + wn * WN + (lane & 31);
    unsigned short* const lo = reinterpret_cast<unsigned short*>(wm ? l2 : l0) + at;
    unsigned short* const hi = reinterpret_cast<unsigned short*>(wm ? l3 : l1) + at;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * (i % HALF) + 8 * (r >> 2) + (r & 3);
                (i < HALF ? lo : hi)[row * BN + 32 * j] = bits(acc[i][j][r]);
            }
    __syncthreads();
    constexpr int vpr = BN / 8;
    const auto flush = [&](const char* l, int q) __attribute__((always_inline)) {
#pragma unroll
        for (int k0 = 0; k0 < Q * vpr; k0 += NT) {
            const int k = k0 + tid, r = k / vpr, c = (k % vpr) * 8;
            if (q * Q + r < rows && c < cols) *reinterpret_cast<u32x4*>(out + (q * Q + r) * ld + c) = *reinterpret_cast<const u32x4*>(l + (r * BN + c) * 2);
        }
    };
    flush(l0, 0);
    __builtin_amdgcn_sched_barrier(0);                         // (not all sixteen vectors in registers beside the accumulators)
    flush(l1, 1);
    __builtin_amdgcn_sched_barrier(0);
    flush(l2, 2);
    __builtin_amdgcn_sched_barrier(0);
    flush(l3, 3);
}

// backward of the logits of one piece: lanes = words, registers = rows
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void ll_dz_kernel(const LossArgs a) {
    typedef TileProduct<typename Term<T>::type, BM, BN, WM, WN, false, false, Term<T>::pairs, true> P;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int NP = Term<T>::planes;
    LL_LDS(BM, BN);
    __shared__ float slse[BM], sw[BM], srow[BM], sdb[BM / WM][BN];
    __shared__ int stg[BM];
    const int count = a.st.count[0], tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5;
    int rt, wt;
    if (!ll_tile((count + BM - 1) / BM, (a.vp + BN - 1) / BN, rt, wt)) return;
    const int m0 = rt * BM, w0 = a.v0 + wt * BN, end = a.v0 + a.vp;
    typename P::A oa;
    typename P::B ob;
    oa.init_rows([&](int r) { return (const char*)(a.xc + (long long)(m0 + r) * NP * a.d.D); }, wave, lane);
    ob.init_rows([&](int r) { return (const char*)a.wp + (long long)min(w0 + r, a.d.V - 1) * NP * a.d.D * 2; }, wave, lane);
    oa.plane = ob.plane = (long long)a.d.D * 2;
    const float top = a.st.sums[1];
    for (int i = tid; i < BM; i += P::NT) {
        const bool ok = m0 + i < count;
        const int row = ok ? a.st.idx[m0 + i] : 0;
        const long long tg = ok ? a.d.target[(row / a.d.T) * a.d.ld_target + row % a.d.T] : -1;
        slse[i] = ok ? a.st.lse[m0 + i] : __builtin_inff();
        sw[i] = ok ? a.d.mask[(row / a.d.T) * a.d.ld_mask + row % a.d.T] / top : 0.f;
        stg[i] = tg >= w0 && tg < min(w0 + BN, end) ? (int)(tg - w0) : -1;
        if (F32) srow[i] = ok ? a.sx[m0 + i] * LOG2E : 0.f;
    }
    f32x16 acc[P::MI][P::NI];
    P::run(acc, oa, ob, 0, (a.d.D + BK - 1) / BK, a.d.D, LL_BUFFERS, wave, lane);
    const int wm = wave / P::NWN, wn = wave % P::NWN;
    float wscale[P::NI], bias[P::NI], sum[P::NI];
    int word[P::NI];
#pragma unroll
    for (int j = 0; j < P::NI; ++j) {
        word[j] = wn * WN + 32 * j + (lane & 31);
        const int v = w0 + word[j];
        bias[j] = v < end ? (a.d.bias ? to_f32(a.d.bias, v, a.d.dtype) * LOG2E : 0.f) : NEG_INF;
        wscale[j] = F32 ? a.sw[min(v, a.d.V - 1)] : 1.f;
        sum[j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < P::MI; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {                         // (rows outside, words inside: what belongs to a row is read once and not kept)
            const int ml = wm * WM + 32 * i + 8 * q + 4 * g;
            const f32x4 l4 = *reinterpret_cast<const f32x4*>(slse + ml), w4 = *reinterpret_cast<const f32x4*>(sw + ml);
            typedef int i32x4 __attribute__((ext_vector_type(4)));
            const i32x4 t4 = *reinterpret_cast<const i32x4*>(stg + ml);
            f32x4 s4 = {LOG2E, LOG2E, LOG2E, LOG2E};
            if (F32) s4 = *reinterpret_cast<const f32x4*>(srow + ml);
#pragma unroll
            for (int j = 0; j < P::NI; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // (f32: the logit rounded as in the forward, so that p is what its denominator holds of it)
                    const float x = acc[i][j][4 * q + e];
                    const float p = __builtin_amdgcn_exp2f(F32 ? fmaf(x, s4[e] * wscale[j], bias[j]) - l4[e] : x * LOG2E + (bias[j] - l4[e]));
                    const float dz = w4[e] == 0.f ? 0.f : (p - (t4[e] == word[j] ? 1.f : 0.f)) * w4[e];
                    acc[i][j][4 * q + e] = dz;
                    sum[j] += dz;
                }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
    for (int j = 0; j < P::NI; ++j) {
        sum[j] += __shfl_xor(sum[j], 32, 64);
        if (g == 0) sdb[wm][word[j]] = sum[j];
    }
    __syncthreads();
    for (int nl = tid; nl < BN; nl += P::NT) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < BM / WM; ++w) s += sdb[w][nl];
        if (wt * BN + nl < a.ldz) a.pdb[(long long)rt * a.ldz + wt * BN + nl] = s;
    }
    const int cols = a.ldz - wt * BN;
    if constexpr (!F32) {
        store_tile<BM, BN, WM, WN, P::MI, P::NI, P::NT>(acc, [&](float v) { return to_bits<T>(v * DzScale<T>::up); }, a.dz + (long long)m0 * a.ldz + wt * BN, a.ldz, BM,
                                                        cols, la0, la1, lb0, lb1, tid, wave, lane);
    } else {
        // Two f16 terms of dz times the weight's scale for dx.  |dz| <= (1 - p_target) |mask| in a row, as far as the rounding of lse (half a
        // unit of |lse| in every p of the row) and of its logarithm lets p sum to one; and |dz| <= |mask|, as no logit is above lse.  That bound
        // is brought to [2^12, 2^13) against the largest weight scale, so that a row decided by one word keeps its small values.  It holds
        // because the logits are the forward's bit for bit; should a matrix unit add in another order for exchanged operands, a value past it
        // is rounding error alone, and is held at the largest f16 (NaN stays NaN).  Then three bf16 terms of dz for dW.  The values are scaled
        // and unscaled by powers of two in place, and hidden from the optimizer between the passes: it would keep every conversion of one
        // pass for the next and spill.
        const float wtop = a.st.sums[2];
        for (int i = tid; i < BM; i += P::NT) {
            float u = 0.f;
            if (m0 + i < count) {
                const float miss = fmaxf(1.f - __builtin_amdgcn_exp2f(a.st.tz[m0 + i] - slse[i]), 0.f) + fmaf(fabsf(slse[i]), 0x1p-24f, 0x1p-21f);
                int e;
                (void)frexpf(fminf(miss, 1.f) * wtop * fabsf(sw[i]), &e);
                u = ldexpf(1.f, max(min(13 - e, 120), -120));
                if (wt == 0) a.up[m0 + i] = 1.f / u;
            }
            srow[i] = u;
        }
        __syncthreads();
        const auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < P::MI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 u4 = *reinterpret_cast<const f32x4*>(srow + wm * WM + 32 * i + 8 * q + 4 * g);
#pragma unroll
                    for (int j = 0; j < P::NI; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = f(acc[i][j][4 * q + e], u4[e], wscale[j]);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
            for (int i = 0; i < P::MI; ++i)
#pragma unroll
                for (int j = 0; j < P::NI; ++j) asm volatile("" : "+v"(acc[i][j]));
        };
        const auto put = [&](auto bits, unsigned short* out, long long ld) __attribute__((always_inline)) {
            store_tile<BM, BN, WM, WN, P::MI, P::NI, P::NT>(acc, bits, out, ld, BM, cols, la0, la1, lb0, lb1, tid, wave, lane);
            __syncthreads();
        };
        unsigned short* f16 = a.dz + (long long)m0 * 2 * a.ldz + wt * BN;
        unsigned short* b16 = a.dzb + (long long)m0 * 3 * a.ldz + wt * BN;
        const auto bf = [](float v) { return to_bits<__bf16>(v); };
        const auto rest = [](float v, float, float) { return v - (float)(__bf16)v; };
        each([](float v, float u, float w) {
            const float x = v * fmaxf(u * w, 0x1p-60f);       // (so far below f16 it is nothing there, but dW takes v back)
            return x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x;
        });
        put([](float v) { return to_bits<_Float16>(v); }, f16, 2ll * a.ldz);
        each([](float v, float, float) { return v; });
        put([](float v) { return to_bits<_Float16>(v - (float)(_Float16)v); }, f16 + a.ldz, 2ll * a.ldz);
        each([](float v, float u, float w) { return v * (1.f / fmaxf(u * w, 0x1p-60f)); });
        put(bf, b16, 3ll * a.ldz);
        each(rest);
        put(bf, b16 + a.ldz, 3ll * a.ldz);
        each(rest);
        put(bf, b16 + 2 * a.ldz, 3ll * a.ldz);
    }
}

// factor that turns sums of stored dz into gradients: dloss / denom * max |mask| / 2^s (no rows: everything is zero)
__device__ __forceinline__ float grad_factor(const LossArgs& a, float up) {
    if (a.st.count[0] == 0) return 0.f;
    return a.d.dloss[0] / (a.d.denom ? a.d.denom[0] : a.st.sums[0]) * a.st.sums[1] / up;
}

// dW = dz^T x of one piece: lanes = features, registers = words
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void ll_dw_kernel(const LossArgs a) {
    // (f32: six products of the exact bf16 terms -- a rare word's whole column of dz is tiny, no row scale serves it)
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int NP = F32 ? 3 : 1;
    typedef TileProduct<std::conditional_t<F32, __bf16, T>, BM, BN, WM, WN, true, true, F32 ? 6 : 1> P;
    LL_LDS(BM, BN);
    const int count = a.st.count[0], tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nm = (a.vp + BM - 1) / BM, nn = (a.d.D + BN - 1) / BN, total = nm * nn * a.splits;
    const int x = blockIdx.x & 7, q = total >> 3, r = total & 7, id = x * q + min(x, r) + (blockIdx.x >> 3);
    const int split = id / (nm * nn), mt = id % (nm * nn) / nn, ntile = id % nn;
    const int m0 = mt * BM, n0 = ntile * BN, kts = (count + BK - 1) / BK, per = (kts + a.splits - 1) / a.splits;
    const int kt0 = min(kts, split * per), kt1 = min(kts, kt0 + per);
    typename P::A oa;
    typename P::B ob;
    oa.init_cols(F32 ? a.dzb : a.dz, (long long)NP * a.ldz, m0, a.ldz, wave, lane);
    ob.init_cols(F32 ? a.xb : a.xc, (long long)NP * a.d.D, n0, a.d.D, wave, lane);
    oa.plane = 2ll * a.ldz;
    ob.plane = 2ll * a.d.D;
    f32x16 acc[P::MI][P::NI];
    P::run(acc, oa, ob, kt0, kt1, kts * BK, LL_BUFFERS, wave, lane);
    if constexpr (!F32) {
        if (a.splits == 1) {
            const float f = grad_factor(a, DzScale<T>::up);
            store_tile<BM, BN, WM, WN, P::MI, P::NI, P::NT>(acc, [&](float v) { return to_bits<T>(v * f); },
                                                            (unsigned short*)a.d.dweight + (long long)(a.v0 + m0) * a.d.D + n0, a.d.D, a.vp - m0, a.d.D - n0, la0, la1, lb0,
                                                            lb1, tid, wave, lane);
            return;
        }
    }
    const int wm = wave / P::NWN, wn = wave % P::NWN, g = lane >> 5;
    const bool direct = F32 && a.splits == 1;
    const float f = direct ? grad_factor(a, 1.f) : 1.f;
    float* out = direct ? (float*)a.d.dweight + (long long)a.v0 * a.d.D : a.pdw + (long long)split * a.ldz * a.d.D;
#pragma unroll
    for (int i = 0; i < P::MI; ++i)
#pragma unroll
        for (int j = 0; j < P::NI; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = m0 + wm * WM + 32 * i + 8 * (e >> 2) + 4 * g + (e & 3), n = n0 + wn * WN + 32 * j + (lane & 31);
                if (m < a.vp && n < a.d.D) out[(long long)m * a.d.D + n] = acc[i][j][e] * f;
            }
}
template <typename T> __global__ __launch_bounds__(256) void ll_dw_sum_kernel(const LossArgs a) {
    const float f = grad_factor(a, DzScale<T>::up);
    const long long n = (long long)a.vp * a.d.D, stride = (long long)a.ldz * a.d.D;
    T* out = (T*)a.d.dweight + (long long)a.v0 * a.d.D;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256ll * gridDim.x) {
        float s = 0.f;
        for (int k = 0; k < a.splits; ++k) s += a.pdw[k * stride + i];
        out[i] = (T)(s * f);
    }
}

// dx partials of one piece: lanes = features, registers = rows; the words of the piece are cut over `splits` workgroups
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void ll_dx_kernel(const LossArgs a) {
    typedef TileProduct<typename Term<T>::type, BM, BN, WM, WN, false, true, Term<T>::pairs> P;
    constexpr int NP = Term<T>::planes;
    LL_LDS(BM, BN);
    const int count = a.st.count[0], tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nm = (count + BM - 1) / BM, nn = (a.d.D + BN - 1) / BN, splits = ll_splits(nm * nn, a.first_vp / BK, a.splits), total = nm * nn * splits;
    if (blockIdx.x == 0 && tid == 0) a.dx_shares[0] = splits;
    if ((int)blockIdx.x >= total) return;
    const int x = blockIdx.x & 7, q = total >> 3, r = total & 7, id = x * q + min(x, r) + (blockIdx.x >> 3);
    const int split = id / (nm * nn), mt = id % (nm * nn) / nn, ntile = id % nn;
    const int m0 = mt * BM, n0 = ntile * BN, kts = (a.vp + BK - 1) / BK, per = (kts + splits - 1) / splits;
    const int kt0 = min(kts, split * per), kt1 = min(kts, kt0 + per);
    typename P::A oa;
    typename P::B ob;
    oa.init_rows([&](int rr) { return (const char*)(a.dz + (long long)(m0 + rr) * NP * a.ldz); }, wave, lane);
    ob.init_cols(a.wp + (long long)a.v0 * NP * a.d.D, (long long)NP * a.d.D, n0, a.d.D, wave, lane);
    oa.plane = 2ll * a.ldz;
    ob.plane = 2ll * a.d.D;
    f32x16 acc[P::MI][P::NI];
    P::run(acc, oa, ob, kt0, kt1, a.vp, LL_BUFFERS, wave, lane);
    const int wm = wave / P::NWN, wn = wave % P::NWN, g = lane >> 5;
    float* out = a.pdx + (long long)split * a.nr * a.d.D;
#pragma unroll
    for (int i = 0; i < P::MI; ++i)
#pragma unroll
        for (int j = 0; j < P::NI; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = m0 + wm * WM + 32 * i + 8 * (e >> 2) + 4 * g + (e & 3), n = n0 + wn * WN + 32 * j + (lane & 31);
                if (m < count && n < a.d.D) {
                    float* o = out + (long long)m * a.d.D + n;
                    *o = a.first ? acc[i][j][e] : *o + acc[i][j][e];
                }
            }
}
// dx rows in place: the sum of the partials, or zeros for a row that does not count
template <typename T> __global__ __launch_bounds__(256) void ll_dx_sum_kernel(const LossArgs a) {
    const int vec = a.d.D / 8, splits = a.dx_shares[0];
    const long long n = (long long)a.d.B * a.d.T * vec;
    const float f0 = grad_factor(a, DzScale<T>::up);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256ll * gridDim.x) {
        const long long row = i / vec;
        const int c = (int)(i % vec) * 8, p = a.st.pos[row];
        const float f = p >= 0 ? (sizeof(T) == 4 ? f0 * a.up[p] : f0) : 0.f;
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (p >= 0)
            for (int k = 0; k < splits; ++k) {
                const f32x4* src = reinterpret_cast<const f32x4*>(a.pdx + ((long long)k * a.nr + p) * a.d.D + c);
                const f32x4 u = src[0], w = src[1];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[e] += u[e];
                    s[4 + e] += w[e];
                }
            }
        if constexpr (sizeof(T) == 4) {
            float* o = (float*)a.d.dx + row * a.d.D + c;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = s[e] * f;
        } else {
            u32x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = to_bits<T>(s[2 * e] * f) | (uint32_t)to_bits<T>(s[2 * e + 1] * f) << 16;
            *reinterpret_cast<u32x4*>((T*)a.d.dx + row * a.d.D + c) = o;
        }
    }
}
// bias gradient: 64 words x 16 strands of row tiles a workgroup
template <typename T> __global__ __launch_bounds__(1024) void ll_db_kernel(const LossArgs a, int BM) {
    __shared__ float part[16][64];
    const int v = blockIdx.x * 64 + (threadIdx.x & 63), k = threadIdx.x >> 6, tiles = (a.st.count[0] + BM - 1) / BM;
    float s = 0.f;
    if (v < a.vp)
        for (int t = k; t < tiles; t += 16) s += a.pdb[(long long)t * a.ldz + v];
    part[k][threadIdx.x & 63] = s;
    __syncthreads();
    if (k || v >= a.vp) return;
    for (int i = 1; i < 16; ++i) s += part[i][threadIdx.x & 63];
    ((T*)a.d.dbias)[a.v0 + v] = (T)(s * grad_factor(a, 1.f));
}

// ---- f32 operands as 16-bit terms.  One wave a row: the compact rows of x (zeros behind them to a multiple of 256), then the rows of the
// weight.  f16: the row times a power of two that brings its largest magnitude to [2^13, 2^14), in two terms; its inverse in sx / sw.
// (rows below 2^-107 are brought less far; the largest finite row takes 2^-114)
__global__ __launch_bounds__(256) void ll_terms_kernel(const LossArgs a, unsigned short* xp, unsigned short* xb, unsigned short* wp, float* sx, float* sw, int nx) {
    const int lane = threadIdx.x & 63, r = blockIdx.x * 4 + (threadIdx.x >> 6), D = a.d.D, count = a.st.count[0], rows = (count + 255) & ~255;
    const bool of_x = r < nx;
    const int v = r - nx;
    if (of_x ? r >= rows : v >= a.d.V) return;
    const bool zero = of_x && r >= count;
    const float* src = of_x ? (const float*)a.d.x + (zero ? 0 : a.st.idx[r]) * a.d.ldx : (const float*)a.d.weight + (long long)v * D;
    float mx = 0.f;
    if (!zero)
        for (int c = 4 * lane; c < D; c += 256) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(src + c);
            mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
        }
    mx = wave_max(mx);
    int e = 0;
    if (mx > 0.f && mx < __builtin_inff()) (void)frexpf(mx, &e);
    e = min(14 - e, 120);
    const float s = ldexpf(1.f, e);
    if (lane == 0) (of_x ? sx[r] : sw[v]) = ldexpf(1.f, -e);
    unsigned short* out = of_x ? xp + (long long)r * 2 * D : wp + (long long)v * 2 * D;
    for (int c = 8 * lane; c < D; c += 512) {
        u32x4 h, l, b0, b1, b2;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t t[5] = {0, 0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const float x = zero ? 0.f : src[c + 2 * k + w], y = x * s, f = (float)(_Float16)y;
                const float q = x - (float)(__bf16)x;
                t[0] |= (uint32_t)to_bits<_Float16>(y) << (16 * w);
                t[1] |= (uint32_t)to_bits<_Float16>(y - f) << (16 * w);
                t[2] |= (uint32_t)to_bits<__bf16>(x) << (16 * w);
                t[3] |= (uint32_t)to_bits<__bf16>(q) << (16 * w);
                t[4] |= (uint32_t)to_bits<__bf16>(q - (float)(__bf16)q) << (16 * w);
            }
            h[k] = t[0]; l[k] = t[1]; b0[k] = t[2]; b1[k] = t[3]; b2[k] = t[4];
        }
        *reinterpret_cast<u32x4*>(out + c) = h;
        *reinterpret_cast<u32x4*>(out + D + c) = l;
        if (of_x && xb) {
            unsigned short* o = xb + (long long)r * 3 * D + c;
            *reinterpret_cast<u32x4*>(o) = b0;
            *reinterpret_cast<u32x4*>(o + D) = b1;
            *reinterpret_cast<u32x4*>(o + 2 * D) = b2;
        }
    }
}
// sums[2] = largest scale of the weight's rows
__global__ __launch_bounds__(1024) void ll_scale_top_kernel(const float* sw, int V, float* out) {
    __shared__ float part[16];
    float m = 0.f;
    for (int v = threadIdx.x; v < V; v += 1024) m = fmaxf(m, sw[v]);
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) m = fmaxf(m, part[w]);
        out[0] = m;
    }
}

// ---- f32 in the other arithmetics: the products are ekaid_gemm_f32, these are the passes around them
__global__ __launch_bounds__(256) void ll_fill_kernel(float* p, long long n, float v) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256ll * gridDim.x) p[i] = v;
}
// running (max, sum) of every row over one more piece of its logits, and the target's logit; one wave per row
__global__ __launch_bounds__(256) void ll32_stats_kernel(const ekaid_linear_loss_t d, State st, const float* z, int ldz, int v0, int vp, float* run, int first, int last) {
    const long long n = (long long)d.B * d.T, row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= n) return;
    const long long b = row / d.T, t = row % d.T;
    const float mask = d.mask[b * d.ld_mask + t];
    if (mask == 0.f) {
        if (lane == 0 && last) st.nll[row] = 0.f;
        return;
    }
    const float* zp = z + row * ldz;
    const float* bias = (const float*)d.bias;
    float m = NEG_INF, l = 0.f;
    for (int v = lane; v < vp; v += 64) {
        const float x = (zp[v] + (bias ? bias[v0 + v] : 0.f)) * LOG2E;
        const float mm = fmaxf(m, x), base = mm == NEG_INF ? 0.f : mm;
        l = l * __builtin_amdgcn_exp2f(m - base) + __builtin_amdgcn_exp2f(x - base);
        m = mm;
    }
    float M = wave_max(m);
    if (!first) M = fmaxf(M, run[2 * row]);
    const float base = M == NEG_INF ? 0.f : M;
    float s = wave_sum(l * __builtin_amdgcn_exp2f(m - base));
    if (lane) return;
    if (!first) s += run[2 * row + 1] * __builtin_amdgcn_exp2f(run[2 * row] - base);
    const long long tg = d.target[b * d.ld_target + t];
    if (first) st.tz[row] = __builtin_nanf("");
    if (tg >= v0 && tg < v0 + vp) st.tz[row] = (zp[tg - v0] + (bias ? bias[tg] : 0.f)) * LOG2E;
    if (last) {
        const float lse = M + __builtin_amdgcn_logf(s);
        st.lse[row] = lse;
        st.nll[row] = (lse - st.tz[row]) * LN2 * mask;
    } else {
        run[2 * row] = M;
        run[2 * row + 1] = s;
    }
}
// logits of one piece -> their gradients, in place; columns vp .. ldz - 1 and rows that do not count become zero
__global__ __launch_bounds__(256) void ll32_dz_kernel(const ekaid_linear_loss_t d, State st, float* z, int ldz, int v0, int vp) {
    const long long n = (long long)d.B * d.T * ldz;
    const float f = d.dloss[0] / (d.denom ? d.denom[0] : st.sums[0]);
    const float* bias = (const float*)d.bias;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256ll * gridDim.x) {
        const long long row = i / ldz, b = row / d.T, t = row % d.T;
        const int v = (int)(i % ldz);
        const float w = d.mask[b * d.ld_mask + t];
        float g = 0.f;
        if (w != 0.f && v < vp) {
            const float p = __builtin_amdgcn_exp2f((z[i] + (bias ? bias[v0 + v] : 0.f)) * LOG2E - st.lse[row]);
            g = (p - (d.target[b * d.ld_target + t] == v0 + v ? 1.f : 0.f)) * (w * f);
        }
        z[i] = g;
    }
}
// x with the rows that do not count zeroed; VEC floats at a time
template <int VEC> __global__ __launch_bounds__(256) void ll32_clean_kernel(const ekaid_linear_loss_t d, float* xc) {
    const int per = d.D / VEC;
    const long long n = (long long)d.B * d.T * per;
    const float* x = (const float*)d.x;
    typedef float vec __attribute__((ext_vector_type(VEC)));
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256ll * gridDim.x) {
        const int row = (int)(i / per), c = (int)(i % per) * VEC;
        vec v = *reinterpret_cast<const vec*>(x + row * d.ldx + c);
        if (d.mask[(row / d.T) * d.ld_mask + row % d.T] == 0.f) v = 0.f;
        *reinterpret_cast<vec*>(xc + (long long)row * d.D + c) = v;
    }
}
// column sums (a bias gradient without the weight's product to ride on): 64 columns x 16 strands of rows a workgroup, fixed order
__global__ __launch_bounds__(1024) void ll32_db_kernel(const float* z, long long n, int vp, int ldz, float* out) {
    __shared__ float part[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), k = threadIdx.x >> 6;
    float s = 0.f;
    if (c < vp)
        for (long long r = k; r < n; r += 16) s += z[r * ldz + c];
    part[k][threadIdx.x & 63] = s;
    __syncthreads();
    if (k || c >= vp) return;
    for (int i = 1; i < 16; ++i) s += part[i][threadIdx.x & 63];
    out[c] = s;
}

// ---- f32, few words: products on the f32 matrix instructions, whole rows of logits in one workgroup, logits kept for the backward
//
// z[row][word] = (x W^T + bias) log2 e, -infinity behind the last word.  A workgroup takes 16 of the rows that count, its waves every fourth 16
// words; lanes read 16 bytes along the width (four matrix instructions), one 64-wide block ahead.  Workgroups start at different blocks: rows
// of the weight a power of two apart share a few channels of the second-level cache, which all workgroups at one block would wait for.
template <int TW> __global__ __launch_bounds__(256) void ll_narrow_fwd_kernel(const ekaid_linear_loss_t d, State st, float* z, int ldz) {
    __shared__ float sm[4][16], sl[4][16], stz[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, kq = lane >> 4;
    const int count = st.count[0], row = blockIdx.x * 16 + j;
    if ((int)blockIdx.x * 16 >= count) return;
    const int rc = st.idx[min(row, count - 1)];
    const float *xp = (const float*)d.x + (long long)rc * d.ldx + 4 * kq, *wp[TW];
#pragma unroll
    for (int u = 0; u < TW; ++u) wp[u] = (const float*)d.weight + (long long)min(16 * (wave + 4 * u) + j, d.V - 1) * d.D + 4 * kq;
    f32x4 acc[TW];
#pragma unroll
    for (int u = 0; u < TW; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 x0[4], x1[4], w0[4][TW], w1[4][TW];
    auto fetch = [&](int k0, f32x4* xf, f32x4 (*wf)[TW]) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k = k0 + 16 * s;
            const bool in = k + 4 * kq < d.D;
            const int o = in ? k : 0;                          // behind the width: zeros (x and the weight alike, an infinite weight is none here)
            xf[s] = *reinterpret_cast<const f32x4*>(xp + (in ? k : -4 * kq));
            if (!in) xf[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < TW; ++u) {
                wf[s][u] = *reinterpret_cast<const f32x4*>(wp[u] + (in ? o : -4 * kq));
                if (!in) wf[s][u] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
    };
    auto multiply = [&](const f32x4* xf, const f32x4 (*wf)[TW]) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int u = 0; u < TW; ++u) acc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[s][u][c], xf[s][c], acc[u], 0, 0, 0);
    };
    const int blocks = (d.D + 63) >> 6, turn = blockIdx.x % blocks;
    auto at = [&](int k) { return 64 * (k + turn < blocks ? k + turn : k + turn - blocks); };
    fetch(at(0), x0, w0);
    for (int k = 0; k < blocks; k += 2) {
        if (k + 1 < blocks) fetch(at(k + 1), x1, w1);
        multiply(x0, w0);
        if (k + 1 >= blocks) break;
        if (k + 2 < blocks) fetch(at(k + 2), x0, w0);
        multiply(x1, w1);
    }
    const long long target = d.target[(rc / d.T) * d.ld_target + rc % d.T];
    const float* bias = (const float*)d.bias;
    float m = NEG_INF, l = 0.f;
#pragma unroll
    for (int u = 0; u < TW; ++u) {
        const int v0 = 16 * (wave + 4 * u) + 4 * kq;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int v = v0 + i;
            acc[u][i] = v < d.V ? (acc[u][i] + (bias ? bias[min(v, d.V - 1)] : 0.f)) * LOG2E : NEG_INF;
            m = fmaxf(m, acc[u][i]);
            if (v == target && v < d.V) stz[j] = acc[u][i];
        }
        if (row < count && v0 < ldz) *reinterpret_cast<f32x4*>(z + (long long)row * ldz + v0) = acc[u];
    }
    if (wave == 0 && kq == 0 && (target < 0 || target >= d.V)) stz[j] = __builtin_nanf("");
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const float base = m == NEG_INF ? 0.f : m;
#pragma unroll
    for (int u = 0; u < TW; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(acc[u][i] - base);
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (kq == 0) {
        sm[wave][j] = m;
        sl[wave][j] = l;
    }
    __syncthreads();
    if (threadIdx.x >= 16 || row >= count) return;
    const float M = fmaxf(fmaxf(sm[0][j], sm[1][j]), fmaxf(sm[2][j], sm[3][j])), B = M == NEG_INF ? 0.f : M;
    float s = 0.f;
    for (int k = 0; k < 4; ++k) s += sl[k][j] * __builtin_amdgcn_exp2f((sm[k][j] == NEG_INF ? 0.f : sm[k][j]) - B);
    const float lse = M + __builtin_amdgcn_logf(s);
    st.lse[row] = lse;
    st.nll[row] = (lse - stz[j]) * LN2 * d.mask[(rc / d.T) * d.ld_mask + rc % d.T];
}

// dz of the rows row0 .. last - 1 (at most ROWS, counted among those that count) from their kept logits into dst[..][stride], zeros behind
// them: 256 / ROWS threads a row, 16 bytes each
template <int ROWS> __device__ __forceinline__ void narrow_dz(const ekaid_linear_loss_t& d, const State& st, const float* z, int ldz, int row0, int last, float f, float* dst, int stride) {
    constexpr int PER = 256 / ROWS;
    const int r = threadIdx.x / PER, c = threadIdx.x % PER, k = min(row0 + r, last - 1), row = st.idx[k];
    const float w = row0 + r < last ? d.mask[(row / d.T) * d.ld_mask + row % d.T] * f : 0.f, lse = st.lse[k];
    const long long target = d.target[(row / d.T) * d.ld_target + row % d.T];
    for (int v = 4 * c; v < ldz; v += 4 * PER) {
        const f32x4 q = *reinterpret_cast<const f32x4*>(z + (long long)k * ldz + v);
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[r * stride + v + i] = row0 + r < last ? (__builtin_amdgcn_exp2f(q[i] - lse) - (target == v + i ? 1.f : 0.f)) * w : 0.f;
    }
}
// Both gradients in one launch.  Workgroups below nx: 16 rows of dx, dz (LDS) times the weight, the waves take the width 2 x 64 apart; and
// zeros for those of 16 rows of x that do not count.  The others: one of `parts` shares of the rows of dz^T x over 64 of the width, 32 rows
// at a time, the waves take the words; shares joined by ll_narrow_sum.
template <int TW> __global__ __launch_bounds__(256, 3) void ll_narrow_bwd_kernel(const ekaid_linear_loss_t d, State st, const float* z, int ldz, int nx, int nd, int parts, float* pdw, float* pdb) {
    __shared__ __attribute__((aligned(16))) float dz[32 * (64 * TW + 16)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, kq = lane >> 4;
    const int count = st.count[0];
    const float f = d.dloss[0] / (d.denom ? d.denom[0] : st.sums[0]);
    if ((int)blockIdx.x < nx) {
        for (int r = 16 * blockIdx.x + wave; r < min(d.B * d.T, 16 * (int)blockIdx.x + 16); r += 4)
            if (st.pos[r] < 0)
                for (int c = 4 * lane; c < d.D; c += 256) *reinterpret_cast<f32x4*>((float*)d.dx + (long long)r * d.D + c) = f32x4{0.f, 0.f, 0.f, 0.f};
        const int r0 = blockIdx.x * 16, stride = ldz + 2;     // (16 rows two words apart in the banks)
        if (r0 >= count) return;
        narrow_dz<16>(d, st, z, ldz, r0, count, f, dz, stride);
        __syncthreads();
        const float* mine = dz + j * stride + kq;
        for (int d0 = 128 * wave; d0 < d.D; d0 += 512) {
            f32x4 acc[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[h][c] = f32x4{0.f, 0.f, 0.f, 0.f};
            const float *wp0 = (const float*)d.weight + min(d0 + 4 * j, d.D - 4), *wp1 = (const float*)d.weight + min(d0 + 64 + 4 * j, d.D - 4);
            f32x4 a0[4][2], a1[4][2];
            auto fetch = [&](int v0, f32x4 (*a)[2]) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const long long o = (long long)min(v0 + 4 * s + kq, d.V - 1) * d.D;
                    a[s][0] = *reinterpret_cast<const f32x4*>(wp0 + o);
                    a[s][1] = *reinterpret_cast<const f32x4*>(wp1 + o);
                }
            };
            auto multiply = [&](int v0, const f32x4 (*a)[2]) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const float g = mine[v0 + 4 * s];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int c = 0; c < 4; ++c) acc[h][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s][h][c], g, acc[h][c], 0, 0, 0);
                }
            };
            fetch(0, a0);
            for (int v0 = 0; v0 < ldz; v0 += 32) {
                if (v0 + 16 < ldz) fetch(v0 + 16, a1);
                multiply(v0, a0);
                if (v0 + 16 >= ldz) break;
                if (v0 + 32 < ldz) fetch(v0 + 32, a0);
                multiply(v0 + 16, a1);
            }
            if (r0 + j >= count) continue;
            float* out = (float*)d.dx + (long long)st.idx[r0 + j] * d.D;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = d0 + 64 * h + 16 * kq + 4 * i;
                    if (c < d.D) *reinterpret_cast<f32x4*>(out + c) = f32x4{acc[h][0][i], acc[h][1][i], acc[h][2][i], acc[h][3][i]};
                }
        }
        return;
    }
    const int q = blockIdx.x - nx, d0 = (q % nd) * 64, part = q / nd, share = ((count + parts - 1) / parts + 31) & ~31, first = min(count, part * share), last = min(count, first + share);
    const int stride = ldz | 16;                               // (four rows half the banks apart)
    const float* xp = (const float*)d.x + min(d0 + 4 * j, d.D - 4);
    f32x4 acc[TW][4];
#pragma unroll
    for (int u = 0; u < TW; ++u)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[u][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
    for (int r0 = first; r0 < last; r0 += 32) {
        f32x4 xf[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) xf[s] = *reinterpret_cast<const f32x4*>(xp + (long long)st.idx[min(r0 + 4 * s + kq, last - 1)] * d.ldx);
        narrow_dz<32>(d, st, z, ldz, r0, last, f, dz, stride);
        __syncthreads();
        if (d0 == 0 && (int)threadIdx.x < ldz)
            for (int r = 0; r < 32; ++r) sum += dz[r * stride + threadIdx.x];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
#pragma unroll
            for (int u = 0; u < TW; ++u) {
                const float g = dz[(4 * s + kq) * stride + min(16 * (wave + 4 * u), ldz - 16) + j];
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[u][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(g, xf[s][c], acc[u][c], 0, 0, 0);
            }
        }
        __syncthreads();
    }
    if (pdb && d0 == 0 && (int)threadIdx.x < ldz) pdb[(long long)part * ldz + threadIdx.x] = sum;
    if (!pdw || d0 + 4 * j >= d.D) return;
#pragma unroll
    for (int u = 0; u < TW; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int v = 16 * (wave + 4 * u) + 4 * kq + i;
            if (v < d.V) *reinterpret_cast<f32x4*>(pdw + ((long long)part * d.V + v) * d.D + d0 + 4 * j) = f32x4{acc[u][0][i], acc[u][1][i], acc[u][2][i], acc[u][3][i]};
        }
}
// parts of dweight (16 bytes a thread) and of dbias (behind them), added in order
__global__ __launch_bounds__(256) void ll_narrow_sum_kernel(const ekaid_linear_loss_t d, const float* pdw, const float* pdb, int ldz, int parts) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, nw = d.dweight ? (long long)d.V * d.D / 4 : 0;
    if (i < nw) {
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int k = 0; k < parts; ++k) s += reinterpret_cast<const f32x4*>(pdw)[k * nw + i];
        if (!((uintptr_t)d.dweight & 15)) reinterpret_cast<f32x4*>(d.dweight)[i] = s;
        else                                                   // (a slot of a flat gradient buffer)
            for (int e = 0; e < 4; ++e) ((float*)d.dweight)[4 * i + e] = s[e];
    } else if (d.dbias && i - nw < d.V) {
        float s = 0.f;
#pragma unroll 8
        for (int k = 0; k < parts; ++k) s += pdb[(long long)k * ldz + (i - nw)];
        ((float*)d.dbias)[i - nw] = s;
    }
}

// ---- host side
// f32 as 16-bit terms through the tile kernels (below 2^31 products of a matrix the few tiles are bound by latency, and ekaid_gemm_f32 with
// its splits is level or ahead)
bool as_terms(const ekaid_linear_loss_t* a) {
    return a->dtype == EKAID_F32 && a->arith == EKAID_GEMM_F16X2 && (double)a->B * a->T * a->V * a->D >= 2147483648.0 && a->D % 8 == 0 && a->ldx % 4 == 0 &&
           !(((uintptr_t)a->x | (uintptr_t)a->weight) & 15);
}
int ll_check(const ekaid_linear_loss_t* a, const char* who) {
    if (!a) { set_error("%s: null descriptor", who); return EKAID_ERR_ARG; }
    if (a->dtype < EKAID_F32 || a->dtype > EKAID_F16) { set_error("%s: dtype %d", who, a->dtype); return EKAID_ERR_ARG; }
    if (a->B < 0 || a->T < 0 || a->D < 1 || a->V < 1 || (long long)a->B * a->T > (1 << 28) || a->V > (1 << 28)) {
        set_error("%s: bad sizes B=%d T=%d D=%d V=%d", who, a->B, a->T, a->D, a->V);
        return EKAID_ERR_ARG;
    }
    if (a->dtype == EKAID_F32 && (a->arith < EKAID_GEMM_F32_MFMA || a->arith > EKAID_GEMM_F16X2)) { set_error("%s: arithmetic %d", who, a->arith); return EKAID_ERR_ARG; }
    // a launch counts its threads in 32 bits: 64 a row (f32; as terms also a word) or 16, 512 a tile of 256 x 256
    const long long n = (long long)a->B * a->T;
    const bool f32 = a->dtype == EKAID_F32, terms = as_terms(a);
    if ((f32 ? n + (terms ? a->V : 0) : n / 4) > (1 << 26) - 512 || ((!f32 || terms) && (n + 255) / 256 * ((a->V + 255ll) / 256) >= (1 << 23))) {
        set_error("%s: %lld rows and %d words are too many for one launch", who, n, a->V);
        return EKAID_ERR_UNSUPPORTED;
    }
    const int al = a->dtype == EKAID_F32 ? 4 : 16;
    if ((uintptr_t)a->state & 15) { set_error("%s: the state must be 16-byte aligned", who); return EKAID_ERR_ARG; }
    if (a->dtype != EKAID_F32 && (a->D % 8 || a->ldx % 8)) { set_error("%s: width %d / row stride %lld must be multiples of 8", who, a->D, a->ldx); return EKAID_ERR_UNSUPPORTED; }
    if (a->ldx < a->D || a->ldx > (1 << 30)) { set_error("%s: row stride %lld", who, a->ldx); return EKAID_ERR_ARG; }
    if (((uintptr_t)a->x | (uintptr_t)a->weight | (uintptr_t)a->dx | (uintptr_t)a->dweight) & (al - 1)) { set_error("%s: operands must be %d-byte aligned", who, al); return EKAID_ERR_ARG; }
    return EKAID_OK;
}
constexpr size_t PIECE_BYTES = size_t(512) << 20;              // dz (or f32 logits) of one piece
size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// Few words (f32): one launch forms the logits, their statistics and the losses, one both gradients, and the logits, no larger than x
// itself, stay in the state.  A rule of sizes alone, since it says what the state holds.  5760 rows (3740 counting) of width 512, 148
// words, against the route through ekaid_gemm_f32 with its 13 launches: kernels 125 -> 71 us (16 rows a workgroup, bound by the latency of
// the second-level cache and of three dependent stages, not by the f32 matrix rate: 5 of the 22 us of the logits, 12 of the gradients' 35).
// Up to 2^30 products of a matrix, where the f32 matrix rate begins to weigh.  Whole calls, this against 257 words on the other route: 5760 x
// 512 x 256 146 / 172 us, 3500 x 1024 x 256 142 / 170, 8000 x 512 x 256 162 / 166, 2000 x 2048 x 256 180 / 173, beyond it 16000 x 512 x 256 287 / 249.
bool few_words(const ekaid_linear_loss_t* a) {
    return a->dtype == EKAID_F32 && a->V <= 256 && ((a->V + 15) & ~15) <= a->D && a->D % 4 == 0 && (double)a->B * a->T * a->V * a->D <= 1073741824.0;
}
size_t kept_offset(const ekaid_linear_loss_t* a) { return (256 + (size_t)a->B * a->T * 20 + 255) & ~size_t(255); }
struct LossPlan {
    int narrow;                    // few words, and operands in whole 16 bytes
    int parts;                     // shares of dW
    int terms;                     // f32 as 16-bit terms through the tile kernels
    int big;                       // 256 x 256 tiles
    long long n, nr;
    int vp, pieces, ldz;           // words a piece
    int sx, sw;                    // splits of dx (at most), dW
    int dx_grid;
    size_t part, dz, xc, pdb, pdx, pdw, total;        // byte offsets
    size_t wp, xb, xscale, wscale, up, dzb;           // f32 terms
    // f32
    size_t z, run, clean, bnd, gws, gws_bytes;
    int bounds;
};
bool f32_bounds(const ekaid_linear_loss_t* a, long long n, int vp) {
    return a->arith == EKAID_GEMM_F16X2 && (double)n * vp * a->D >= 6e9 && a->D % 4 == 0 && a->ldx % 4 == 0 && std::min({(long long)a->D, n, (long long)vp}) >= 32 &&
           !(((uintptr_t)a->x | (uintptr_t)a->weight) & 15);
}
ekaid_gemm_t product(const float* A, const float* B, float* C, int M, int N, int K, int lda, int ldb, int ldc, int tA, int tB) {
    ekaid_gemm_t g = {};
    g.A = A; g.B = B; g.C = C;
    g.M = M; g.N = N; g.K = K;
    g.lda = lda; g.ldb = ldb; g.ldc = ldc;
    g.transA = tA; g.transB = tB;
    g.batch1 = g.batch2 = 1;
    g.alpha = 1.f;
    g.rdiv = 1;
    return g;
}
LossPlan loss_plan(const ekaid_linear_loss_t* a, int backward) {
    LossPlan p = {};
    p.n = (long long)a->B * a->T;
    p.nr = (p.n + 255) & ~255ll;
    size_t o = 0;
    p.narrow = few_words(a) && a->ldx % 4 == 0 && !(((uintptr_t)a->x | (uintptr_t)a->weight) & 15);
    if (p.narrow) {
        p.ldz = (a->V + 15) & ~15;
        p.parts = (int)std::max(1ll, std::min<long long>(320 / std::max(1, std::min(320, cdiv(a->D, 64))), (p.n + 63) / 64));        // about 320 workgroups, 64 rows or more each
        p.pdw = o; o += backward ? up256((size_t)p.parts * a->V * a->D * 4) : 0;
        p.pdb = o; o += backward ? up256((size_t)p.parts * p.ldz * 4) : 0;
        p.total = o;
        return p;
    }
    p.terms = as_terms(a);
    if (a->dtype == EKAID_F32 && !p.terms) {
        long long vp = (long long)(PIECE_BYTES / 4) / std::max(1ll, p.n);
        vp = std::max(256ll, vp & ~255ll);
        p.vp = (int)std::min<long long>(a->V, vp);
        p.pieces = cdiv(a->V, p.vp);
        p.ldz = (p.vp + 3) & ~3;
        p.bounds = f32_bounds(a, p.n, p.vp);
        p.z = o; o += up256((size_t)p.n * p.ldz * 4);
        p.run = o; o += backward ? 0 : up256((size_t)p.n * 8);
        p.clean = o; o += backward ? up256((size_t)p.n * a->D * 4) : 0;
        // bounds: rows of x, rows of W, columns of x, columns of W, rows and columns of dz
        p.bnd = o; o += p.bounds ? up256(((size_t)2 * p.n + a->V + 2 * a->D + p.ldz + 64) * 4) : 0;
        p.gws = o;
        ekaid_gemm_t g[3] = {product(nullptr, nullptr, nullptr, (int)p.n, p.vp, a->D, (int)a->ldx, a->D, p.ldz, 0, 1),
                             product(nullptr, nullptr, nullptr, (int)p.n, a->D, p.vp, p.ldz, a->D, a->D, 0, 0),
                             product(nullptr, nullptr, nullptr, p.vp, a->D, (int)p.n, p.ldz, a->D, a->D, 1, 0)};
        const int rest = a->V - (p.pieces - 1) * p.vp;
        static float probe;
        for (int k = 0; k < (p.n == 0 ? 0 : backward ? 3 : 1); ++k)
            for (int last = 0; last < 2; ++last) {
                if (last) (k == 0 ? g[k].N : k == 1 ? g[k].K : g[k].M) = rest;
                for (int b = 0; b <= p.bounds; ++b) {
                    g[k].a_amax = g[k].b_amax = b ? &probe : nullptr;
                    g[k].a_rowsum = k == 2 ? &probe : nullptr;
                    p.gws_bytes = std::max(p.gws_bytes, ekaid_gemm_workspace_bytes(&g[k]));
                }
            }
        o += up256(p.gws_bytes);
        p.total = o;
        return p;
    }
    // Tiles of 256 x 256 from half a round of the chip on, counted with all rows (how many count is known on the device alone).  128 / 256 wide,
    // us, forward and gradients, every row counting: f32 1024 x 1024 x 4096 (64 tiles) 325 / 398, x 7936 (124) 585 / 493, 2048 x 1024 x 8192
    // (256) 1093 / 695; bf16 1024 x 1024 x 4096 117 / 166 or more (host-bound), x 8192 (128) 182 / 182, 2048 x 1024 x 8192 316 / 220.
    p.big = (p.nr / 256) * (long long)cdiv(a->V, 256) >= 128;
    const int bt = p.big ? 256 : 128;
    if (p.terms) {
        p.wp = o; o += up256((size_t)a->V * a->D * 4);
        p.wscale = o; o += up256((size_t)a->V * 4);
        p.xscale = o; o += up256((size_t)p.nr * 4);
        p.xc = o; o += up256((size_t)p.nr * a->D * 4);
        p.xb = o; o += backward ? up256((size_t)p.nr * a->D * 6) : 0;
        p.up = o; o += backward ? up256((size_t)p.nr * 4) : 0;
    }
    if (!backward) {
        p.part = o; o += up256((size_t)cdiv(a->V, bt) * p.nr * 8);
        p.total = o;
        return p;
    }
    const int per = p.terms ? 10 : 2;      // bytes of dz a logit
    long long vp = (long long)(PIECE_BYTES / per) / std::max(1ll, p.nr);
    vp = std::max(1024ll, vp & ~255ll);
    p.pieces = cdiv(a->V, std::min<long long>(a->V, vp));
    p.vp = (int)std::min<long long>(a->V, ((a->V + p.pieces - 1) / p.pieces + 255) & ~255);          // even pieces
    p.pieces = cdiv(a->V, p.vp);
    p.ldz = ((p.vp + 63) & ~63) + 64;      // (rows a power of two apart would meet in the same memory channels)
    const size_t dx_bytes = (size_t)p.nr * a->D * 4;
    p.sx = (int)std::max<size_t>(1, std::min<size_t>(16, (size_t(1) << 29) / std::max<size_t>(1, dx_bytes)));
    p.sw = ll_splits(cdiv(p.vp, bt) * cdiv(a->D, bt), (int)(p.nr / BK) * (p.terms ? 6 : 1), 32);
    p.dz = o; o += up256((size_t)p.nr * p.ldz * (p.terms ? 4 : 2));
    p.dzb = o; o += p.terms ? up256((size_t)p.nr * p.ldz * 6) : 0;
    if (!p.terms) { p.xc = o; o += up256((size_t)p.nr * a->D * 2); }
    p.pdb = o; o += up256((size_t)(p.nr / bt) * p.ldz * 4);
    p.pdx = o; o += up256((size_t)p.sx * p.nr * a->D * 4);
    p.pdw = o; o += p.sw > 1 ? up256((size_t)p.sw * p.ldz * a->D * 4) : 0;
    p.total = o + 256;
    const int nn = cdiv(a->D, bt);
    for (int nm = 1; nm <= p.nr / bt; ++nm) p.dx_grid = std::max(p.dx_grid, nm * nn * ll_splits(nm * nn, p.vp / BK, p.sx));      // for any number of rows
    return p;
}
int blocks(long long n) { return (int)std::max(1ll, std::min<long long>((n + 255) / 256, 8192)); }

int fwd32(const ekaid_linear_loss_t* a, const LossPlan& p, State st, char* ws, hipStream_t s) {
    float* z = (float*)(ws + p.z);
    float* xr = (float*)(ws + p.bnd);
    float* wr = xr + ((p.n + 3) & ~3ll);
    if (p.bounds) {
        const long long nb = ((p.n + 3) & ~3ll) + a->V;
        hipLaunchKernelGGL(ll_fill_kernel, dim3(blocks(nb)), dim3(256), 0, s, xr, nb, 0.f);
        if (int rc = ekaid_amax_rc((const float*)a->x, p.n, a->D, (int)a->ldx, xr, nullptr, 1, s)) return rc;
        if (int rc = ekaid_amax_rc((const float*)a->weight, a->V, a->D, a->D, wr, nullptr, 1, s)) return rc;
    }
    for (int k = 0; k < p.pieces; ++k) {
        const int v0 = k * p.vp, vp = std::min(p.vp, a->V - v0);
        ekaid_gemm_t g = product((const float*)a->x, (const float*)a->weight + (size_t)v0 * a->D, z, (int)p.n, vp, a->D, (int)a->ldx, a->D, p.ldz, 0, 1);
        if (p.bounds) { g.a_amax = xr; g.b_amax = wr + v0; }
        if (int rc = ekaid_gemm_f32(&g, ws + p.gws, p.gws_bytes, s)) return rc;
        hipLaunchKernelGGL(ll32_stats_kernel, dim3(cdiv(p.n, 4)), dim3(256), 0, s, *a, st, z, p.ldz, v0, vp, (float*)(ws + p.run), k == 0, k == p.pieces - 1);
    }
    return check_launch("linear_loss_fwd");
}
int bwd32(const ekaid_linear_loss_t* a, const LossPlan& p, State st, char* ws, hipStream_t s) {
    float* z = (float*)(ws + p.z);
    float* xc = (float*)(ws + p.clean);
    float* xr = (float*)(ws + p.bnd);
    const long long n4 = (p.n + 3) & ~3ll, v4 = (a->V + 3) & ~3;
    float *wr = xr + n4, *xcol = wr + v4, *wcol = xcol + ((a->D + 3) & ~3), *zr = wcol + ((a->D + 3) & ~3), *zcol = zr + n4;
    if (a->D % 4 == 0 && a->ldx % 4 == 0 && !((uintptr_t)a->x & 15)) hipLaunchKernelGGL(ll32_clean_kernel<4>, dim3(blocks(p.n * (a->D / 4))), dim3(256), 0, s, *a, xc);
    else hipLaunchKernelGGL(ll32_clean_kernel<1>, dim3(blocks(p.n * a->D)), dim3(256), 0, s, *a, xc);
    if (a->dbias) hipLaunchKernelGGL(ll_fill_kernel, dim3(blocks(a->V)), dim3(256), 0, s, (float*)a->dbias, (long long)a->V, 0.f);
    if (p.bounds) {
        hipLaunchKernelGGL(ll_fill_kernel, dim3(blocks(zr - xr)), dim3(256), 0, s, xr, (long long)(zr - xr), 0.f);
        if (int rc = ekaid_amax_rc(xc, p.n, a->D, a->D, xr, xcol, 1, s)) return rc;
        if (int rc = ekaid_amax_rc((const float*)a->weight, a->V, a->D, a->D, wr, wcol, 1, s)) return rc;
    }
    for (int k = 0; k < p.pieces; ++k) {
        const int v0 = k * p.vp, vp = std::min(p.vp, a->V - v0), vz = (vp + 3) & ~3;
        const float* W = (const float*)a->weight + (size_t)v0 * a->D;
        // the SAME product as in the forward (same operand, same plan): probabilities sum to one as the forward's denominator says
        ekaid_gemm_t g = product((const float*)a->x, W, z, (int)p.n, vp, a->D, (int)a->ldx, a->D, p.ldz, 0, 1);
        if (p.bounds) { g.a_amax = xr; g.b_amax = wr + v0; }
        if (int rc = ekaid_gemm_f32(&g, ws + p.gws, p.gws_bytes, s)) return rc;
        hipLaunchKernelGGL(ll32_dz_kernel, dim3(blocks(p.n * p.ldz)), dim3(256), 0, s, *a, st, z, p.ldz, v0, vp);
        if (p.bounds) {
            const long long nz = n4 + p.ldz;
            hipLaunchKernelGGL(ll_fill_kernel, dim3(blocks(nz)), dim3(256), 0, s, zr, nz, 0.f);
            if (int rc = ekaid_amax_rc(z, p.n, vz, p.ldz, zr, zcol, 1, s)) return rc;
        }
        if (a->dx) {
            g = product(z, W, (float*)a->dx, (int)p.n, a->D, vp, p.ldz, a->D, a->D, 0, 0);
            g.accumulate = k > 0;
            if (p.bounds) { g.a_amax = zr; g.b_amax = wcol; }
            if (int rc = ekaid_gemm_f32(&g, ws + p.gws, p.gws_bytes, s)) return rc;
        }
        if (a->dweight) {
            g = product(z, xc, (float*)a->dweight + (size_t)v0 * a->D, vp, a->D, (int)p.n, p.ldz, a->D, a->D, 1, 0);
            if (a->dbias) g.a_rowsum = (float*)a->dbias + v0;
            if (p.bounds) { g.a_amax = zcol; g.b_amax = xcol; }
            if (int rc = ekaid_gemm_f32(&g, ws + p.gws, p.gws_bytes, s)) return rc;
        } else if (a->dbias) {
            hipLaunchKernelGGL(ll32_db_kernel, dim3(cdiv(vp, 64)), dim3(1024), 0, s, z, p.n, vp, p.ldz, (float*)a->dbias + v0);
        }
    }
    return check_launch("linear_loss_bwd");
}

template <int TW> int narrow(const ekaid_linear_loss_t* a, const LossPlan& p, State st, char* ws, bool backward, hipStream_t s) {
    float* z = (float*)((char*)a->state + kept_offset(a));
    if (!backward) {
        hipLaunchKernelGGL(ll_narrow_fwd_kernel<TW>, dim3(cdiv(p.n, 16)), dim3(256), 0, s, *a, st, z, p.ldz);
        return check_launch("linear_loss_fwd");
    }
    float *pdw = a->dweight ? (float*)(ws + p.pdw) : nullptr, *pdb = a->dbias ? (float*)(ws + p.pdb) : nullptr;
    const int nx = a->dx ? cdiv(p.n, 16) : 0, nd = a->dweight ? cdiv(a->D, 64) : 1, nw = a->dweight || a->dbias ? nd * p.parts : 0;
    if (nx + nw) hipLaunchKernelGGL(ll_narrow_bwd_kernel<TW>, dim3(nx + nw), dim3(256), 0, s, *a, st, z, p.ldz, nx, nd, p.parts, pdw, pdb);
    if (nw) hipLaunchKernelGGL(ll_narrow_sum_kernel, dim3(cdiv((a->dweight ? (long long)a->V * a->D / 4 : 0) + a->V, 256)), dim3(256), 0, s, *a, pdw, pdb, p.ldz, p.parts);
    return check_launch("linear_loss_bwd");
}
int narrow(const ekaid_linear_loss_t* a, const LossPlan& p, State st, char* ws, bool backward, hipStream_t s) {
    switch (cdiv(a->V, 64)) {
        case 1: return narrow<1>(a, p, st, ws, backward, s);
        case 2: return narrow<2>(a, p, st, ws, backward, s);
        case 3: return narrow<3>(a, p, st, ws, backward, s);
        default: return narrow<4>(a, p, st, ws, backward, s);
    }
}

void launch_terms(const LossArgs& a, const LossPlan& p, hipStream_t s) {
    hipLaunchKernelGGL(ll_terms_kernel, dim3(cdiv(p.nr + a.d.V, 4)), dim3(256), 0, s, a, (unsigned short*)a.xc, (unsigned short*)a.xb, (unsigned short*)a.wp, (float*)a.sx,
                       (float*)a.sw, (int)p.nr);
    if (a.xb) hipLaunchKernelGGL(ll_scale_top_kernel, dim3(1), dim3(1024), 0, s, a.sw, a.d.V, a.st.sums + 2);
}
template <typename T, int BT, int WM, int WN> int fwd16(LossArgs a, const LossPlan& p, hipStream_t s) {
    constexpr int NT = (BT / WM) * (BT / WN) * 64;
    const int tiles = cdiv(a.d.V, BT);
    if constexpr (sizeof(T) == 4) launch_terms(a, p, s);
    hipLaunchKernelGGL((ll_stats_kernel<T, BT, BT, WM, WN>), dim3((int)(p.nr / BT) * tiles), dim3(NT), 0, s, a);
    hipLaunchKernelGGL(ll_lse_kernel, dim3(cdiv(p.n, 64)), dim3(1024), 0, s, a, tiles);
    return check_launch("linear_loss_fwd");
}
template <typename T, int BT, int WM, int WN> int bwd16(LossArgs a, const LossPlan& p, hipStream_t s) {
    constexpr int NT = (BT / WM) * (BT / WN) * 64;
    const ekaid_linear_loss_t& d = a.d;
    const int rt = (int)(p.nr / BT), dt = cdiv(d.D, BT);
    if constexpr (sizeof(T) == 4) launch_terms(a, p, s);
    else hipLaunchKernelGGL(ll_gather_kernel, dim3(blocks(p.nr * (d.D / 8))), dim3(256), 0, s, a, (unsigned short*)a.xc);
    for (int k = 0; k < p.pieces; ++k) {
        a.v0 = k * p.vp;
        a.vp = std::min(p.vp, d.V - a.v0);
        a.first = k == 0;
        hipLaunchKernelGGL((ll_dz_kernel<T, BT, BT, WM, WN>), dim3(rt * cdiv(a.vp, BT)), dim3(NT), 0, s, a);
        if (d.dweight) {
            a.splits = p.sw;
            hipLaunchKernelGGL((ll_dw_kernel<T, BT, BT, WM, WN>), dim3(cdiv(a.vp, BT) * dt * p.sw), dim3(NT), 0, s, a);
            if (p.sw > 1) hipLaunchKernelGGL(ll_dw_sum_kernel<T>, dim3(blocks((long long)a.vp * d.D)), dim3(256), 0, s, a);
        }
        if (d.dbias) hipLaunchKernelGGL(ll_db_kernel<T>, dim3(cdiv(a.vp, 64)), dim3(1024), 0, s, a, BT);
        if (d.dx) {
            a.splits = p.sx;
            hipLaunchKernelGGL((ll_dx_kernel<T, BT, BT, WM, WN>), dim3(p.dx_grid), dim3(NT), 0, s, a);
        }
    }
    a.splits = p.sx;
    if (d.dx) hipLaunchKernelGGL(ll_dx_sum_kernel<T>, dim3(blocks(p.n * (d.D / 8))), dim3(256), 0, s, a);
    return check_launch("linear_loss_bwd");
}
LossArgs loss_args(const ekaid_linear_loss_t* a, const LossPlan& p, char* ws, bool backward) {
    LossArgs k = {};
    k.d = *a;
    k.st = state_of(a->state, p.n);
    k.nr = p.nr;
    k.vp = k.first_vp = p.vp;
    k.ldz = p.ldz;
    k.part = (float2*)(ws + p.part);
    k.dz = (unsigned short*)(ws + p.dz);
    k.xc = (const unsigned short*)(ws + p.xc);
    k.wp = (const unsigned short*)a->weight;
    if (p.terms) {
        k.wp = (const unsigned short*)(ws + p.wp);
        k.sx = (const float*)(ws + p.xscale);
        k.sw = (const float*)(ws + p.wscale);
        k.xb = backward ? (const unsigned short*)(ws + p.xb) : nullptr;
        k.up = (float*)(ws + p.up);
        k.dzb = (unsigned short*)(ws + p.dzb);
    }
    k.pdb = (float*)(ws + p.pdb);
    k.pdx = (float*)(ws + p.pdx);
    k.dx_shares = (int*)(ws + p.total - 256);
    k.pdw = (float*)(ws + p.pdw);
    return k;
}
}  // namespace
}  // namespace ekaid

extern "C" size_t ekaid_linear_loss_state_bytes(const ekaid_linear_loss_t* a) {
    if (ekaid::ll_check(a, "linear_loss_state_bytes")) return 0;
    return ekaid::kept_offset(a) + (ekaid::few_words(a) ? (size_t)a->B * a->T * ((a->V + 15) & ~15) * 4 : 0);
}
extern "C" size_t ekaid_linear_loss_workspace_bytes(const ekaid_linear_loss_t* a, int backward) {
    if (ekaid::ll_check(a, "linear_loss_workspace_bytes")) return 0;
    const ekaid::GemmModeScope mode(a->arith);             // (what ekaid_gemm_f32 needs depends on it)
    return ekaid::loss_plan(a, backward).total;
}
extern "C" int ekaid_linear_loss_fwd(const ekaid_linear_loss_t* a, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace ekaid;
    if (int rc = ll_check(a, "linear_loss_fwd")) return rc;
    if (!a->loss || !a->state || !a->weight || (a->B * (long long)a->T && (!a->x || !a->target || !a->mask))) { set_error("linear_loss_fwd: null operand"); return EKAID_ERR_ARG; }
    const GemmModeScope mode(a->arith);
    const LossPlan p = loss_plan(a, 0);
    if (workspace_bytes < p.total || (p.total && !workspace)) { set_error("linear_loss_fwd: workspace of %zu bytes needed", p.total); return EKAID_ERR_ARG; }
    hipStream_t s = (hipStream_t)stream;
    const State st = state_of(a->state, p.n);
    hipLaunchKernelGGL(ll_rows_kernel, dim3(1), dim3(1024), 0, s, a->mask, a->ld_mask, a->B, a->T, st);
    int rc = check_launch("linear_loss_fwd");
    if (rc == EKAID_OK && p.n) {
        if (p.narrow) rc = narrow(a, p, st, (char*)workspace, false, s);
        else if (a->dtype == EKAID_F32 && !p.terms) rc = fwd32(a, p, st, (char*)workspace, s);
        else {
            const LossArgs k = loss_args(a, p, (char*)workspace, false);
            if (a->dtype == EKAID_F32) rc = p.big ? fwd16<float, 256, 128, 64>(k, p, s) : fwd16<float, 128, 64, 64>(k, p, s);
            else if (a->dtype == EKAID_BF16) rc = p.big ? fwd16<__bf16, 256, 128, 64>(k, p, s) : fwd16<__bf16, 128, 64, 64>(k, p, s);
            else rc = p.big ? fwd16<_Float16, 256, 128, 64>(k, p, s) : fwd16<_Float16, 128, 64, 64>(k, p, s);
        }
    }
    if (rc) return rc;
    hipLaunchKernelGGL(ll_loss_kernel, dim3(1), dim3(1024), 0, s, *a, st, a->dtype == EKAID_F32 && !p.terms && !p.narrow);
    return check_launch("linear_loss_fwd");
}
extern "C" int ekaid_linear_loss_bwd(const ekaid_linear_loss_t* a, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace ekaid;
    if (int rc = ll_check(a, "linear_loss_bwd")) return rc;
    const GemmModeScope mode(a->arith);                    // (the forward's, whatever the device's mode has become)
    const LossPlan p = loss_plan(a, 1);
    if (p.n == 0) { set_error("linear_loss_bwd: no rows (the caller zeroes the gradients)"); return EKAID_ERR_ARG; }
    if (!a->dloss || !a->state || !a->x || !a->weight || !a->target || !a->mask) { set_error("linear_loss_bwd: null operand"); return EKAID_ERR_ARG; }
    if (workspace_bytes < p.total || !workspace) { set_error("linear_loss_bwd: workspace of %zu bytes needed", p.total); return EKAID_ERR_ARG; }
    hipStream_t s = (hipStream_t)stream;
    if (p.narrow && ((uintptr_t)a->dx & 15)) { set_error("linear_loss_bwd: dx must be 16-byte aligned"); return EKAID_ERR_ARG; }
    if (p.narrow) return narrow(a, p, state_of(a->state, p.n), (char*)workspace, true, s);
    if (a->dtype == EKAID_F32 && !p.terms) return bwd32(a, p, state_of(a->state, p.n), (char*)workspace, s);
    const LossArgs k = loss_args(a, p, (char*)workspace, true);
    if (a->dtype == EKAID_F32) return p.big ? bwd16<float, 256, 128, 64>(k, p, s) : bwd16<float, 128, 64, 64>(k, p, s);
    if (a->dtype == EKAID_BF16) return p.big ? bwd16<__bf16, 256, 128, 64>(k, p, s) : bwd16<__bf16, 128, 64, 64>(k, p, s);
    return p.big ? bwd16<_Float16, 256, 128, 64>(k, p, s) : bwd16<_Float16, 128, 64, 64>(k, p, s);
}
