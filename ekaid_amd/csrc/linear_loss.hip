// Vocabulary loss of a linear layer without its logits, and its gradient (include/ekaid_hip.h: ekaid_linear_loss_t).
//
// 16-bit types: the rows that count (mask != 0) are listed once; products run on tiles of 256 x 256 x 64 (128 x 128 x 64 when the grid
// would not fill the chip), operands copied to LDS without passing registers, one tile ahead of the matrix instructions.
//   forward   z^T = W x^T per tile -> per-row maximum and sum of the tile's words; a second small kernel joins the tiles
//   backward  per piece of the vocabulary: z again -> dz = (softmax - onehot) mask, rounded to the type, and the bias partials;
//             dW = dz^T x;  dx partials += dz W.   Three products where the formula has three, one more than if logits were kept: at width D
//             forming z again costs 2 D flops a logit, reading a kept f32 one and writing it 8 bytes.
// f32: the same pieces around ekaid_gemm_f32 (its arithmetic: the two-term f16 or the exact three-term bf16 split).
#include "common.h"
#include "../../include/ekaid_hip.h"
#include <algorithm>

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

// ---- per-call state: [meta: count | sum mask | max |mask| ...][lse2 N][target logit N][idx N][pos N]
struct State {
    int* count;
    float* sums;         // [0] sum of the mask, [1] max |mask|
    float* lse;          // log2 denominators, by compact row (16-bit) or by row (f32)
    float* tz;           // target logit in powers of two
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
    s.idx = (int*)(s.tz + n);
    s.pos = s.idx + n;
    return s;
}

// the rows that count, in order; sum and largest magnitude of the mask.  One workgroup: thread t owns a run of rows (fixed order).
__global__ __launch_bounds__(1024) void ll_rows_kernel(const float* mask, long long ld, int B, int T, State st) {
    const long long n = (long long)B * T;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const long long per = (n + 1023) / 1024, r0 = min(n, t * per), r1 = min(n, r0 + per);
    int c = 0;
    float s = 0.f, mx = 0.f;
    for (long long r = r0; r < r1; ++r) {
        const float m = mask[(r / T) * ld + r % T];
        c += m != 0.f ? 1 : 0;
        s += m;
        mx = fmaxf(mx, fabsf(m));
    }
    int incl = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(incl, o, 64);
        if (lane >= o) incl += v;
    }
    __shared__ int wsum[16];
    __shared__ float ssum[1024], smax[16];
    ssum[t] = s;
    mx = wave_max(mx);
    if (lane == 63) wsum[wave] = incl;
    if (lane == 0) smax[wave] = mx;
    __syncthreads();
    int base = incl - c, total = 0;
    for (int w = 0; w < 16; ++w) {
        if (w < wave) base += wsum[w];
        total += wsum[w];
    }
    for (long long r = r0; r < r1; ++r) {
        const bool on = mask[(r / T) * ld + r % T] != 0.f;
        if (on) {
            st.idx[base] = (int)r;
            st.tz[base] = __builtin_nanf("");                  // stays NaN when the target is no word of the vocabulary
        }
        st.pos[r] = on ? base++ : -1;
    }
    for (int w = 512; w > 0; w >>= 1) {
        if (t < w) ssum[t] += ssum[t + w];
        __syncthreads();
    }
    if (t == 0) {
        float m = smax[0];
        for (int w = 1; w < 16; ++w) m = fmaxf(m, smax[w]);
        st.count[0] = total;
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
//   contracted index contiguous (COL = false): LDS [R][64], the 16-byte slots of row r permuted by ^ (r & 7);
//   contracted index strided   (COL = true):  LDS [64][R], the 64-byte groups of row k permuted by ^ (k & 3)
// -- so that fragment reads meet few bank conflicts; the permutation is applied to the GLOBAL address, LDS is written in lane order.
template <int R, bool COL, int NW> struct Operand {
    static constexpr int chunks = R / (8 * NW);
    const char* p[chunks];
    int k0[chunks];                       // first contracted element of this lane's vector (COL: its row), or a large value: read zeros
    long long step;                       // bytes per 64 contracted elements
    __device__ __forceinline__ void issue(char* lds, int kt, int K, int wave) const {
#pragma unroll
        for (int i = 0; i < chunks; ++i) {
            const char* src = kt * BK + k0[i] < K ? p[i] + kt * step : (const char*)zero16;
            __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)(lds + (i * NW + wave) * 1024), 16, 0, 0);
        }
    }
    // row(r): address of row r's first element (any valid address for rows that do not exist)
    template <typename F> __device__ __forceinline__ void init_rows(F row, int wave, int lane) {
        static_assert(!COL, "");
        step = BK * 2;
#pragma unroll
        for (int i = 0; i < chunks; ++i) {
            const int r = (i * NW + wave) * 8 + (lane >> 3), s = (lane & 7) ^ (r & 7);
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
        return *reinterpret_cast<const u32x4*>(lds + r * 128 + (((c * 2 + g) ^ (r & 7)) << 4));
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

// acc[mi][ni] += sum over k in [64 kt0, 64 kt1) of A(m, k) B(n, k); BM x BN per workgroup, WM x WN per wave.  Two LDS buffers: the copies
// of tile t + 1 are under way while tile t is multiplied; ONE barrier a tile, behind a wait for this wave's copies and LDS reads.
template <typename T, int BM, int BN, int WM, int WN, bool ACOL, bool BCOL> struct TileProduct {
    static constexpr int NWN = BN / WN, NW = (BM / WM) * NWN, NT = 64 * NW, MI = WM / 32, NI = WN / 32;
    typedef Operand<BM, ACOL, NW> A;
    typedef Operand<BN, BCOL, NW> B;
    static __device__ __forceinline__ void settle() {
        __builtin_amdgcn_s_waitcnt(0x0070);               // vmcnt 0, lgkmcnt 0
        __builtin_amdgcn_s_barrier();
    }
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
    // K: contracted elements in all (vectors beyond read as zero)
    static __device__ __forceinline__ void run(f32x16 (&acc)[MI][NI], const A& oa, const B& ob, int kt0, int kt1, int K, char* a0, char* a1, char* b0, char* b1,
                                               int wave, int lane) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
        if (kt0 < kt1) {
            oa.issue(a0, kt0, K, wave);
            ob.issue(b0, kt0, K, wave);
        }
        for (int kt = kt0; kt < kt1; kt += 2) {
            settle();
            if (kt + 1 < kt1) {
                oa.issue(a1, kt + 1, K, wave);
                ob.issue(b1, kt + 1, K, wave);
            }
            step(acc, a0, b0, wave, lane);
            if (kt + 1 < kt1) {
                settle();
                if (kt + 2 < kt1) {
                    oa.issue(a0, kt + 2, K, wave);
                    ob.issue(b0, kt + 2, K, wave);
                }
                step(acc, a1, b1, wave, lane);
            }
        }
        settle();                                           // the LDS is free for the epilogue
    }
};
#define LL_LDS(BM, BN)                                                                                                          \
    __shared__ __attribute__((aligned(16))) char la0[BM * BK * 2], la1[BM * BK * 2], lb0[BN * BK * 2], lb1[BN * BK * 2]

struct LossArgs {
    ekaid_linear_loss_t d;
    State st;
    long long nr;             // rows of the compact buffers (multiple of 256)
    int row_tiles;            // upper bound of row tiles (grid)
    int v0, vp;               // first word and words of this piece; ldz = leading dimension of dz
    int ldz;
    float2* part;             // [word tiles][nr] per-row (max, sum) of a tile
    unsigned short* dz;       // [nr][ldz]
    const unsigned short* xc; // [nr][D] the rows that count, zeros behind
    float* pdb;               // [row tiles][ldz] bias partials
    float* pdx;               // [splits][nr][D]
    float* pdw;               // [splits][ldz][D] (splits > 1)
    int splits;
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
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void ll_stats_kernel(const LossArgs a) {
    typedef TileProduct<T, BM, BN, WM, WN, false, false> P;
    LL_LDS(BM, BN);
    const int count = a.st.count[0], tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5;
    int rt, wt;
    if (!ll_tile((count + BN - 1) / BN, (a.d.V + BM - 1) / BM, rt, wt)) return;
    const int w0 = wt * BM, n0 = rt * BN;
    typename P::A oa;
    typename P::B ob;
    oa.init_rows([&](int r) { return (const char*)a.d.weight + (long long)min(w0 + r, a.d.V - 1) * a.d.D * 2; }, wave, lane);
    ob.init_rows([&](int r) { return (const char*)a.d.x + a.st.idx[min(n0 + r, count - 1)] * a.d.ldx * 2; }, wave, lane);
    f32x16 acc[P::MI][P::NI];
    P::run(acc, oa, ob, 0, (a.d.D + BK - 1) / BK, a.d.D, la0, la1, lb0, lb1, wave, lane);
    float* bias = reinterpret_cast<float*>(la0);               // [BM], -inf behind the vocabulary
    float2* red = reinterpret_cast<float2*>(la1);              // [BM / WM][BN]
    for (int i = tid; i < BM; i += P::NT) bias[i] = w0 + i < a.d.V ? (a.d.bias ? to_f32(a.d.bias, w0 + i, a.d.dtype) * LOG2E : 0.f) : NEG_INF;
    __syncthreads();
    const int wm = wave / P::NWN, wn = wave % P::NWN;
#pragma unroll
    for (int j = 0; j < P::NI; ++j) {
        const int nl = wn * WN + 32 * j + (lane & 31), n = n0 + nl;
        const bool ok = n < count;
        const int row = ok ? a.st.idx[n] : 0;
        const long long tg = ok ? a.d.target[(row / a.d.T) * a.d.ld_target + row % a.d.T] : -1;
        const int tl = tg >= w0 && tg < w0 + BM && tg < a.d.V ? (int)(tg - w0) : -1;
        float mx = NEG_INF, tz = 0.f;
        bool mine = false;
#pragma unroll
        for (int i = 0; i < P::MI; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int ml = wm * WM + 32 * i + 8 * q + 4 * g;
                const f32x4 b4 = *reinterpret_cast<const f32x4*>(bias + ml);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float z = acc[i][j][4 * q + e] * LOG2E + b4[e];
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

// lse of a row from its tiles: 64 rows x 4 strands of tiles a workgroup
__global__ __launch_bounds__(256) void ll_lse_kernel(const LossArgs a, int tiles) {
    __shared__ float sm[4][64], sl[4][64];
    const int r = threadIdx.x & 63, k = threadIdx.x >> 6;
    const long long n = (long long)blockIdx.x * 64 + r;
    const bool ok = n < a.st.count[0];
    float m = NEG_INF, l = 0.f;
    if (ok)
        for (int t = k; t < tiles; t += 4) {
            const float2 p = a.part[t * a.nr + n];
            const float mm = fmaxf(m, p.x), base = mm == NEG_INF ? 0.f : mm;
            l = l * __builtin_amdgcn_exp2f(m - base) + p.y * __builtin_amdgcn_exp2f(p.x - base);
            m = mm;
        }
    sm[k][r] = m;
    sl[k][r] = l;
    __syncthreads();
    if (k || !ok) return;
    for (int i = 1; i < 4; ++i) m = fmaxf(m, sm[i][r]);
    const float base = m == NEG_INF ? 0.f : m;
    l = 0.f;
    for (int i = 0; i < 4; ++i) l += sl[i][r] * __builtin_amdgcn_exp2f(sm[i][r] - base);
    a.st.lse[n] = m + __builtin_amdgcn_logf(l);
}

// loss = sum mask (lse - z_target) / denom, in double and a fixed order
__global__ __launch_bounds__(1024) void ll_loss_kernel(const ekaid_linear_loss_t d, State st, int by_row) {
    __shared__ double s[1024];
    const int count = by_row ? d.B * d.T : st.count[0];
    double x = 0.0;
    for (int n = threadIdx.x; n < count; n += 1024) {
        const int row = by_row ? n : st.idx[n];
        const float m = d.mask[(row / d.T) * d.ld_mask + row % d.T];
        if (m != 0.f) x += (double)((st.lse[n] - st.tz[n]) * LN2) * m;
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

// output tile through LDS: lanes hold columns, registers rows; written as whole 16-byte vectors
template <typename T, int BM, int BN, int WM, int WN, int MI, int NI, int NT>
__device__ __forceinline__ void store_tile(const f32x16 (&acc)[MI][NI], float f, T* out, long long ld, int rows, int cols, char* l0, char* l1, char* l2, char* l3,
                                           int tid, int wave, int lane) {
    constexpr int NWN = BN / WN, Q = BM / 4;                   // a quarter of the rows in each of the four operand buffers
    static_assert(Q * BN <= BM * BK && Q % 32 == 0, "");
    const int wm = wave / NWN, wn = wave % NWN, g = lane >> 5;
    char* const buf[4] = {l0, l1, l2, l3};
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int rb = wm * WM + 32 * i;
        unsigned short* t = reinterpret_cast<unsigned short*>(buf[rb / Q]) + (rb % Q) * BN;
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) t[(8 * (r >> 2) + 4 * g + (r & 3)) * BN + wn * WN + 32 * j + (lane & 31)] = to_bits<T>(acc[i][j][r] * f);
    }
    __syncthreads();
    constexpr int vpr = BN / 8;
    for (int k = tid; k < BM * vpr; k += NT) {
        const int r = k / vpr, c = (k % vpr) * 8;
        if (r < rows && c < cols) *reinterpret_cast<u32x4*>(out + r * ld + c) = *reinterpret_cast<const u32x4*>(buf[r / Q] + ((r % Q) * BN + c) * 2);
    }
}

// backward of the logits of one piece: lanes = words, registers = rows
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void ll_dz_kernel(const LossArgs a) {
    typedef TileProduct<T, BM, BN, WM, WN, false, false> P;
    LL_LDS(BM, BN);
    __shared__ float slse[BM], sw[BM], sdb[BM / WM][BN];
    __shared__ int stg[BM];
    const int count = a.st.count[0], tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5;
    int rt, wt;
    if (!ll_tile((count + BM - 1) / BM, (a.vp + BN - 1) / BN, rt, wt)) return;
    const int m0 = rt * BM, w0 = a.v0 + wt * BN, end = a.v0 + a.vp;
    typename P::A oa;
    typename P::B ob;
    oa.init_rows([&](int r) { return (const char*)(a.xc + (long long)(m0 + r) * a.d.D); }, wave, lane);
    ob.init_rows([&](int r) { return (const char*)a.d.weight + (long long)min(w0 + r, a.d.V - 1) * a.d.D * 2; }, wave, lane);
    const float top = a.st.sums[1];
    for (int i = tid; i < BM; i += P::NT) {
        const bool ok = m0 + i < count;
        const int row = ok ? a.st.idx[m0 + i] : 0;
        const long long tg = ok ? a.d.target[(row / a.d.T) * a.d.ld_target + row % a.d.T] : -1;
        slse[i] = ok ? a.st.lse[m0 + i] : __builtin_inff();
        sw[i] = ok ? a.d.mask[(row / a.d.T) * a.d.ld_mask + row % a.d.T] / top : 0.f;
        stg[i] = tg >= w0 && tg < min(w0 + BN, end) ? (int)(tg - w0) : -1;
    }
    f32x16 acc[P::MI][P::NI];
    P::run(acc, oa, ob, 0, (a.d.D + BK - 1) / BK, a.d.D, la0, la1, lb0, lb1, wave, lane);
    const int wm = wave / P::NWN, wn = wave % P::NWN;
#pragma unroll
    for (int j = 0; j < P::NI; ++j) {
        const int nl = wn * WN + 32 * j + (lane & 31), v = w0 + nl;
        const float bias = v < end ? (a.d.bias ? to_f32(a.d.bias, v, a.d.dtype) * LOG2E : 0.f) : NEG_INF;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < P::MI; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int ml = wm * WM + 32 * i + 8 * q + 4 * g;
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(slse + ml), w4 = *reinterpret_cast<const f32x4*>(sw + ml);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(acc[i][j][4 * q + e] * LOG2E + bias - l4[e]);
                    const float dz = w4[e] == 0.f ? 0.f : (p - (stg[ml + e] == nl ? 1.f : 0.f)) * w4[e];
                    acc[i][j][4 * q + e] = dz;
                    sum += dz;
                }
            }
        sum += __shfl_xor(sum, 32, 64);
        if (g == 0) sdb[wm][nl] = sum;
    }
    __syncthreads();
    for (int nl = tid; nl < BN; nl += P::NT) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < BM / WM; ++w) s += sdb[w][nl];
        if (wt * BN + nl < a.ldz) a.pdb[(long long)rt * a.ldz + wt * BN + nl] = s;
    }
    store_tile<T, BM, BN, WM, WN, P::MI, P::NI, P::NT>(acc, DzScale<T>::up, (T*)a.dz + (long long)m0 * a.ldz + wt * BN, a.ldz, BM, a.ldz - wt * BN, la0, la1, lb0, lb1, tid,
                                                       wave, lane);
}

// factor that turns sums of stored dz into gradients: dloss / denom * max |mask| / 2^s (no rows: everything is zero)
__device__ __forceinline__ float grad_factor(const LossArgs& a, float up) {
    if (a.st.count[0] == 0) return 0.f;
    return a.d.dloss[0] / (a.d.denom ? a.d.denom[0] : a.st.sums[0]) * a.st.sums[1] / up;
}

// dW = dz^T x of one piece: lanes = features, registers = words
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void ll_dw_kernel(const LossArgs a) {
    typedef TileProduct<T, BM, BN, WM, WN, true, true> P;
    LL_LDS(BM, BN);
    const int count = a.st.count[0], tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nm = (a.vp + BM - 1) / BM, nn = (a.d.D + BN - 1) / BN, total = nm * nn * a.splits;
    const int x = blockIdx.x & 7, q = total >> 3, r = total & 7, id = x * q + min(x, r) + (blockIdx.x >> 3);
    const int split = id / (nm * nn), mt = id % (nm * nn) / nn, ntile = id % nn;
    const int m0 = mt * BM, n0 = ntile * BN, kts = (count + BK - 1) / BK, per = (kts + a.splits - 1) / a.splits;
    const int kt0 = min(kts, split * per), kt1 = min(kts, kt0 + per);
    typename P::A oa;
    typename P::B ob;
    oa.init_cols(a.dz, a.ldz, m0, a.ldz, wave, lane);
    ob.init_cols(a.xc, a.d.D, n0, a.d.D, wave, lane);
    f32x16 acc[P::MI][P::NI];
    P::run(acc, oa, ob, kt0, kt1, kts * BK, la0, la1, lb0, lb1, wave, lane);
    if (a.splits == 1) {
        store_tile<T, BM, BN, WM, WN, P::MI, P::NI, P::NT>(acc, grad_factor(a, DzScale<T>::up), (T*)a.d.dweight + (long long)(a.v0 + m0) * a.d.D + n0, a.d.D, a.vp - m0,
                                                           a.d.D - n0, la0, la1, lb0, lb1, tid, wave, lane);
        return;
    }
    const int wm = wave / P::NWN, wn = wave % P::NWN, g = lane >> 5;
    float* out = a.pdw + (long long)split * a.ldz * a.d.D;
#pragma unroll
    for (int i = 0; i < P::MI; ++i)
#pragma unroll
        for (int j = 0; j < P::NI; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = m0 + wm * WM + 32 * i + 8 * (e >> 2) + 4 * g + (e & 3), n = n0 + wn * WN + 32 * j + (lane & 31);
                if (m < a.vp && n < a.d.D) out[(long long)m * a.d.D + n] = acc[i][j][e];
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
    typedef TileProduct<T, BM, BN, WM, WN, false, true> P;
    LL_LDS(BM, BN);
    const int count = a.st.count[0], tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nm = (count + BM - 1) / BM, nn = (a.d.D + BN - 1) / BN, total = nm * nn * a.splits;
    if ((int)blockIdx.x >= total) return;
    const int x = blockIdx.x & 7, q = total >> 3, r = total & 7, id = x * q + min(x, r) + (blockIdx.x >> 3);
    const int split = id / (nm * nn), mt = id % (nm * nn) / nn, ntile = id % nn;
    const int m0 = mt * BM, n0 = ntile * BN, kts = (a.vp + BK - 1) / BK, per = (kts + a.splits - 1) / a.splits;
    const int kt0 = min(kts, split * per), kt1 = min(kts, kt0 + per);
    typename P::A oa;
    typename P::B ob;
    oa.init_rows([&](int rr) { return (const char*)(a.dz + (long long)(m0 + rr) * a.ldz); }, wave, lane);
    ob.init_cols((const unsigned short*)a.d.weight + (long long)a.v0 * a.d.D, a.d.D, n0, a.d.D, wave, lane);
    f32x16 acc[P::MI][P::NI];
    P::run(acc, oa, ob, kt0, kt1, a.vp, la0, la1, lb0, lb1, wave, lane);
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
    const int vec = a.d.D / 8;
    const long long n = (long long)a.d.B * a.d.T * vec;
    const float f0 = grad_factor(a, DzScale<T>::up);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256ll * gridDim.x) {
        const long long row = i / vec;
        const int c = (int)(i % vec) * 8, p = a.st.pos[row];
        const float f = p >= 0 ? f0 : 0.f;
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (p >= 0)
            for (int k = 0; k < a.splits; ++k) {
                const f32x4* src = reinterpret_cast<const f32x4*>(a.pdx + ((long long)k * a.nr + p) * a.d.D + c);
                const f32x4 u = src[0], w = src[1];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[e] += u[e];
                    s[4 + e] += w[e];
                }
            }
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = to_bits<T>(s[2 * e] * f) | (uint32_t)to_bits<T>(s[2 * e + 1] * f) << 16;
        *reinterpret_cast<u32x4*>((T*)a.d.dx + row * a.d.D + c) = o;
    }
}
template <typename T> __global__ __launch_bounds__(256) void ll_db_kernel(const LossArgs a, int BM) {
    const int v = blockIdx.x * 256 + threadIdx.x, tiles = (a.st.count[0] + BM - 1) / BM;
    if (v >= a.vp) return;
    float s = 0.f;
    for (int t = 0; t < tiles; ++t) s += a.pdb[(long long)t * a.ldz + v];
    ((T*)a.d.dbias)[a.v0 + v] = (T)(s * grad_factor(a, 1.f));
}

// ---- f32: the products are ekaid_gemm_f32, these are the passes around them
__global__ __launch_bounds__(256) void ll_fill_kernel(float* p, long long n, float v) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256ll * gridDim.x) p[i] = v;
}
// running (max, sum) of every row over one more piece of its logits, and the target's logit; one wave per row
__global__ __launch_bounds__(256) void ll32_stats_kernel(const ekaid_linear_loss_t d, State st, const float* z, int ldz, int v0, int vp, float* run, int first, int last) {
    const long long n = (long long)d.B * d.T, row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= n) return;
    const long long b = row / d.T, t = row % d.T;
    if (d.mask[b * d.ld_mask + t] == 0.f) return;
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
    if (last) st.lse[row] = M + __builtin_amdgcn_logf(s);
    else {
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
__global__ __launch_bounds__(256) void ll32_clean_kernel(const ekaid_linear_loss_t d, float* xc) {
    const long long n = (long long)d.B * d.T * d.D;
    const float* x = (const float*)d.x;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256ll * gridDim.x) {
        const long long row = i / d.D;
        xc[i] = d.mask[(row / d.T) * d.ld_mask + row % d.T] == 0.f ? 0.f : x[row * d.ldx + i % d.D];
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

// ---- host side
int ll_check(const ekaid_linear_loss_t* a, const char* who) {
    if (!a) { set_error("%s: null descriptor", who); return EKAID_ERR_ARG; }
    if (a->dtype < EKAID_F32 || a->dtype > EKAID_F16) { set_error("%s: dtype %d", who, a->dtype); return EKAID_ERR_ARG; }
    if (a->B < 0 || a->T < 0 || a->D < 1 || a->V < 1 || (long long)a->B * a->T > (1 << 28) || a->V > (1 << 28)) {
        set_error("%s: bad sizes B=%d T=%d D=%d V=%d", who, a->B, a->T, a->D, a->V);
        return EKAID_ERR_ARG;
    }
    const int al = a->dtype == EKAID_F32 ? 4 : 16;
    if (a->dtype != EKAID_F32 && (a->D % 8 || a->ldx % 8)) { set_error("%s: width %d / row stride %lld must be multiples of 8", who, a->D, a->ldx); return EKAID_ERR_UNSUPPORTED; }
    if (a->ldx < a->D || a->ldx > (1 << 30)) { set_error("%s: row stride %lld", who, a->ldx); return EKAID_ERR_ARG; }
    if (((uintptr_t)a->x | (uintptr_t)a->weight | (uintptr_t)a->dx | (uintptr_t)a->dweight) & (al - 1)) { set_error("%s: operands must be %d-byte aligned", who, al); return EKAID_ERR_ARG; }
    return EKAID_OK;
}
constexpr size_t PIECE_BYTES = size_t(256) << 20;              // dz (or f32 logits) of one piece: what the 256 MB last-level cache can hold
size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

struct LossPlan {
    int big;                       // 256 x 256 tiles
    long long n, nr;
    int vp, pieces, ldz;           // words a piece
    int sx, sw;                    // splits of dx, dW
    size_t part, dz, xc, pdb, pdx, pdw, total;        // byte offsets
    // f32
    size_t z, run, clean, bnd, gws, gws_bytes;
    int bounds;
};
bool f32_bounds(const ekaid_linear_loss_t* a, long long n, int vp) {
    return gemm_mode() == EKAID_GEMM_F16X2 && (double)n * vp * a->D >= 6e9 && a->D % 4 == 0 && a->ldx % 4 == 0 && std::min({(long long)a->D, n, (long long)vp}) >= 32 &&
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
    if (a->dtype == EKAID_F32) {
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
    p.big = (p.nr / 256) * (long long)cdiv(a->V, 256) >= 128;
    const int bt = p.big ? 256 : 128;
    if (!backward) {
        p.part = o; o += up256((size_t)cdiv(a->V, bt) * p.nr * 8);
        p.total = o;
        return p;
    }
    long long vp = (long long)(PIECE_BYTES / 2) / std::max(1ll, p.nr);
    vp = std::max(1024ll, vp & ~255ll);
    p.pieces = cdiv(a->V, std::min<long long>(a->V, vp));
    p.vp = (int)std::min<long long>(a->V, ((a->V + p.pieces - 1) / p.pieces + 255) & ~255);          // even pieces
    p.pieces = cdiv(a->V, p.vp);
    p.ldz = (p.vp + 63) & ~63;
    auto split = [](long long tiles, int ksteps) {
        long long s = tiles >= 192 ? 1 : (256 + tiles - 1) / std::max(1ll, tiles);
        return (int)std::max(1ll, std::min<long long>(s, ksteps / 8));
    };
    p.sx = split(p.nr / bt * cdiv(a->D, bt), p.vp / BK);
    p.sw = split((long long)cdiv(p.vp, bt) * cdiv(a->D, bt), (int)(p.nr / BK));
    p.dz = o; o += up256((size_t)p.nr * p.ldz * 2);
    p.xc = o; o += up256((size_t)p.nr * a->D * 2);
    p.pdb = o; o += up256((size_t)(p.nr / bt) * p.ldz * 4);
    p.pdx = o; o += up256((size_t)p.sx * p.nr * a->D * 4);
    p.pdw = o; o += p.sw > 1 ? up256((size_t)p.sw * p.ldz * a->D * 4) : 0;
    p.total = o;
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
    hipLaunchKernelGGL(ll32_clean_kernel, dim3(blocks(p.n * a->D)), dim3(256), 0, s, *a, xc);
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

template <typename T, int BT, int WM, int WN> int fwd16(LossArgs a, const LossPlan& p, hipStream_t s) {
    constexpr int NT = (BT / WM) * (BT / WN) * 64;
    const int tiles = cdiv(a.d.V, BT);
    hipLaunchKernelGGL((ll_stats_kernel<T, BT, BT, WM, WN>), dim3((int)(p.nr / BT) * tiles), dim3(NT), 0, s, a);
    hipLaunchKernelGGL(ll_lse_kernel, dim3(cdiv(p.n, 64)), dim3(256), 0, s, a, tiles);
    return check_launch("linear_loss_fwd");
}
template <typename T, int BT, int WM, int WN> int bwd16(LossArgs a, const LossPlan& p, hipStream_t s) {
    constexpr int NT = (BT / WM) * (BT / WN) * 64;
    const ekaid_linear_loss_t& d = a.d;
    const int rt = (int)(p.nr / BT), dt = cdiv(d.D, BT);
    hipLaunchKernelGGL(ll_gather_kernel, dim3(blocks(p.nr * (d.D / 8))), dim3(256), 0, s, a, (unsigned short*)a.xc);
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
        if (d.dbias) hipLaunchKernelGGL(ll_db_kernel<T>, dim3(cdiv(a.vp, 256)), dim3(256), 0, s, a, BT);
        if (d.dx) {
            a.splits = p.sx;
            hipLaunchKernelGGL((ll_dx_kernel<T, BT, BT, WM, WN>), dim3(rt * dt * p.sx), dim3(NT), 0, s, a);
        }
    }
    a.splits = p.sx;
    if (d.dx) hipLaunchKernelGGL(ll_dx_sum_kernel<T>, dim3(blocks(p.n * (d.D / 8))), dim3(256), 0, s, a);
    return check_launch("linear_loss_bwd");
}
LossArgs loss_args(const ekaid_linear_loss_t* a, const LossPlan& p, char* ws) {
    LossArgs k = {};
    k.d = *a;
    k.st = state_of(a->state, p.n);
    k.nr = p.nr;
    k.vp = p.vp;
    k.ldz = p.ldz;
    k.part = (float2*)(ws + p.part);
    k.dz = (unsigned short*)(ws + p.dz);
    k.xc = (const unsigned short*)(ws + p.xc);
    k.pdb = (float*)(ws + p.pdb);
    k.pdx = (float*)(ws + p.pdx);
    k.pdw = (float*)(ws + p.pdw);
    return k;
}
}  // namespace
}  // namespace ekaid

extern "C" size_t ekaid_linear_loss_state_bytes(const ekaid_linear_loss_t* a) {
    if (ekaid::ll_check(a, "linear_loss_state_bytes")) return 0;
    return 256 + (size_t)a->B * a->T * 16;
}
extern "C" size_t ekaid_linear_loss_workspace_bytes(const ekaid_linear_loss_t* a, int backward) {
    if (ekaid::ll_check(a, "linear_loss_workspace_bytes")) return 0;
    return ekaid::loss_plan(a, backward).total;
}
extern "C" int ekaid_linear_loss_fwd(const ekaid_linear_loss_t* a, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace ekaid;
    if (int rc = ll_check(a, "linear_loss_fwd")) return rc;
    if (!a->loss || !a->state || !a->weight || (a->B * (long long)a->T && (!a->x || !a->target || !a->mask))) { set_error("linear_loss_fwd: null operand"); return EKAID_ERR_ARG; }
    const LossPlan p = loss_plan(a, 0);
    if (workspace_bytes < p.total || (p.total && !workspace)) { set_error("linear_loss_fwd: workspace of %zu bytes needed", p.total); return EKAID_ERR_ARG; }
    hipStream_t s = (hipStream_t)stream;
    const State st = state_of(a->state, p.n);
    hipLaunchKernelGGL(ll_rows_kernel, dim3(1), dim3(1024), 0, s, a->mask, a->ld_mask, a->B, a->T, st);
    int rc = check_launch("linear_loss_fwd");
    if (rc == EKAID_OK && p.n) {
        if (a->dtype == EKAID_F32) rc = fwd32(a, p, st, (char*)workspace, s);
        else {
            const LossArgs k = loss_args(a, p, (char*)workspace);
            if (a->dtype == EKAID_BF16) rc = p.big ? fwd16<__bf16, 256, 128, 64>(k, p, s) : fwd16<__bf16, 128, 64, 64>(k, p, s);
            else rc = p.big ? fwd16<_Float16, 256, 128, 64>(k, p, s) : fwd16<_Float16, 128, 64, 64>(k, p, s);
        }
    }
    if (rc) return rc;
    hipLaunchKernelGGL(ll_loss_kernel, dim3(1), dim3(1024), 0, s, *a, st, a->dtype == EKAID_F32);
    return check_launch("linear_loss_fwd");
}
extern "C" int ekaid_linear_loss_bwd(const ekaid_linear_loss_t* a, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace ekaid;
    if (int rc = ll_check(a, "linear_loss_bwd")) return rc;
    const LossPlan p = loss_plan(a, 1);
    if (p.n == 0) { set_error("linear_loss_bwd: no rows (the caller zeroes the gradients)"); return EKAID_ERR_ARG; }
    if (!a->dloss || !a->state || !a->x || !a->weight || !a->target || !a->mask) { set_error("linear_loss_bwd: null operand"); return EKAID_ERR_ARG; }
    if (workspace_bytes < p.total || !workspace) { set_error("linear_loss_bwd: workspace of %zu bytes needed", p.total); return EKAID_ERR_ARG; }
    hipStream_t s = (hipStream_t)stream;
    if (a->dtype == EKAID_F32) return bwd32(a, p, state_of(a->state, p.n), (char*)workspace, s);
    const LossArgs k = loss_args(a, p, (char*)workspace);
    if (a->dtype == EKAID_BF16) return p.big ? bwd16<__bf16, 256, 128, 64>(k, p, s) : bwd16<__bf16, 128, 64, 64>(k, p, s);
    return p.big ? bwd16<_Float16, 256, 128, 64>(k, p, s) : bwd16<_Float16, 128, 64, 64>(k, p, s);
}
