// Forward of the attention operators (include/ekaid_hip.h: ekaid_attn_t): one pass over the keys with the running maximum and sum.
#include "attn.h"
#include <algorithm>

namespace ekaid {

template <int G, int NB>
__device__ __forceinline__ void drop_scores(const AttnArgs& a, typename Blk<G>::acc (&s)[NB], int b, int h, int i, int j0, int lane) {
    constexpr int ng = Blk<G>::ng, nq = Blk<G>::nq;
    const uint64_t seed = drop_seed_value(a.seed);
#pragma unroll
    for (int q = 0; q < NB * nq; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[q / nq][4 * (q % nq) + e] *= drop_kept(a, seed, b, h, i, j0 + 4 * ng * q + 4 * (lane / G) + e);
}

template <typename T, int DH, int G>
__device__ __forceinline__ void write_rows(const AttnArgs& a, const RowWork& w, typename Blk<G>::acc (&o)[DH / G], float m, float l, int i, int h,
                                           bool ok, int lane) {
    constexpr int ng = Blk<G>::ng, nq = Blk<G>::nq;
    const int g = lane / G;
    l = across_groups_sum<G>(l);
    if (!ok) return;
    const long long row = ((long long)w.b * a.d.H + h) * a.d.Lq + i;
    if (a.splits > 1) {
        const long long rows = (long long)a.d.B * a.d.H * a.d.Lq;
        float* p = a.po + (w.split * rows + row) * a.d.dh;
#pragma unroll
        for (int q = 0; q < DH / G * nq; ++q) {
            const int col = 4 * ng * q + 4 * g;
            const auto& t = o[q / nq];
            if (col < a.d.dh) store4<float>(p + col, t[4 * (q % nq)], t[4 * (q % nq) + 1], t[4 * (q % nq) + 2], t[4 * (q % nq) + 3]);
        }
        if (g == 0) {
            a.pml[2 * (w.split * rows + row)] = m;
            a.pml[2 * (w.split * rows + row) + 1] = l;
        }
        return;
    }
    const float inv = l == 0.f ? 0.f : a.inv_keep / l;
    T* p = reinterpret_cast<T*>(a.d.out) + ((long long)w.b * a.d.Lq + i) * a.d.H * a.d.dh + (long long)h * a.d.dh;
#pragma unroll
    for (int q = 0; q < DH / G * nq; ++q) {
        const int col = 4 * ng * q + 4 * g;
        const auto& t = o[q / nq];
        if (col < a.d.dh) {
            const float x0 = t[4 * (q % nq)] * inv, x1 = t[4 * (q % nq) + 1] * inv, x2 = t[4 * (q % nq) + 2] * inv, x3 = t[4 * (q % nq) + 3] * inv;
            store4<T>(p + col, x0, x1, x2, x3);
            if (sizeof(T) == 2 && a.d.out32) store4<float>(a.d.out32 + (p - reinterpret_cast<T*>(a.d.out)) + col, x0, x1, x2, x3);
        }
    }
    if (g == 0 && a.d.lse) a.d.lse[row] = l == 0.f ? POS_INF : m + __builtin_amdgcn_logf(l);
}

// ---- few query rows (a new token; the heads that share keys packed into the rows): 16 rows a workgroup, its NW waves take blocks of keys in
// turn and are joined at the end.  Nothing is shared before that: keys go from memory to registers as fragments; f32 values likewise (a
// lane's four columns of a row are its element of four output blocks: columns 64 x + 4 n + t are row n of block 4 x + t), 16-bit values
// through a buffer of the wave for the transposing read.  One block ahead is under way while a block is worked on.  Bound by reading the
// keys and values once: 16 x 32 heads of 128 on 8, up to 8192 keys, bf16 (361 MB): 77 us, 4.7 TB/s, and 4.6 us for the join of its splits;
// 32 x 16 heads of 64, up to 4096 keys with a bias table, f16 (355 MB): 83 us, 4.3 TB/s; 64 x 4 heads of 256, up to 104 keys, f32 (36 MB): 16 us.
template <typename T, int DH> struct FewBlock {
    static constexpr int KB = sizeof(T) == 4 ? 16 : 32, NB = KB / 16, NC = DH / (Elem<T>::epl * 4), NV = sizeof(T) == 4 ? 4 * (DH / 64) : 0;
    u32x4 k[NB][NC], v[NV + 1];
    uint32_t ok[NB];                       // bit i: key i of the block may be attended
    TileCopy<T, DH, KB, 1> copy;           // (16-bit values)
    __device__ __forceinline__ void load(const ekaid_attn_t& d, const T* kb, const T* vb, const unsigned char* mask, int j0, int end, T* vs, int lane) {
        const int n = lane & 15, g = lane >> 4;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int j = j0 + 16 * b + n;
            const bool valid = j < end && (!mask || mask[j]);
            ok[b] = (uint32_t)__ballot(valid) & 0xffffu;
            const T* row = kb + (long long)j * d.k_row;
#pragma unroll
            for (int c = 0; c < NC; ++c) k[b][c] = row_frag_global<T, 16>(row, c, d.dh, valid, lane);
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool valid = (ok[0] >> (4 * g + e)) & 1;
                const T* row = vb + (long long)(j0 + 4 * g + e) * d.v_row;
#pragma unroll
                for (int x = 0; x < DH / 64; ++x) {
                    u32x4 z = {0u, 0u, 0u, 0u};
                    if (valid && 64 * x + 4 * n < d.dh) z = *reinterpret_cast<const u32x4*>(row + 64 * x + 4 * n);
                    v[e * (DH / 64) + x] = z;
                }
            }
        } else {
            uint32_t bits = ok[0];
            if constexpr (NB > 1) bits |= ok[1] << 16;
#pragma unroll
            for (int i = 0; i < TileCopy<T, DH, KB, 1>::chunks; ++i) {
                const int cr = i * TileCopy<T, DH, KB, 1>::per, row = cr + copy.lrow, s = copy.p ^ swz<T, DH>(row);
                const char* src = copy.lane_base + (long long)(j0 + cr) * copy.stride + s * 16;
                src = ((bits >> row) & 1) && s * Elem<T>::epl < d.dh ? src : (const char*)attn_zero16;
                __builtin_amdgcn_global_load_lds((global_void)src, (lds_void)(reinterpret_cast<char*>(vs) + i * 1024), 16, 0, 0);
            }
        }
    }
};

template <typename T, int DH, int NW>
__global__ __launch_bounds__(64 * NW, sizeof(T) * DH >= 512 ? 1 : 2) void attn_few_kernel(const AttnArgs a) {
    typedef FewBlock<T, DH> Block;
    constexpr int NT = 64 * NW, NB = Block::NB, NC = Block::NC, KB = Block::KB, MT = DH / 16, nv16 = sizeof(T) == 4 ? 4 : KB * DH;
    __shared__ __attribute__((aligned(16))) T va[NW][nv16], vb_[NW][nv16];
    __shared__ float sml[NW][2][16];
    extern __shared__ __attribute__((aligned(16))) char smem[];
    // [NW][rows][DH] outputs of the waves, 4-column groups permuted by row; 16-bit: over the value buffers, whose work is done by then
    float* join = sizeof(T) == 4 ? reinterpret_cast<float*>(smem) : reinterpret_cast<float*>(va);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, n = lane & 15;
    const RowWork w(a);
    const ekaid_attn_t& d = a.d;
    const int R = d.Lq * a.gp, row0 = w.tile * 16, rows = min(16, R - row0), r = min(row0 + n, R - 1);
    const bool ok = n < rows;
    float* bias = reinterpret_cast<float*>(smem) + (sizeof(T) == 4 ? NW * rows * DH : 0);
    const int i = r / a.gp, hg = r % a.gp, h = w.head0 + hg;
    const int p0 = query_pos(d, w.b), pos = p0 + i, len = key_len(d, w.b);
    const int kend = d.causal ? max(0, min(len, p0 + (row0 + rows - 1) / a.gp + 1)) : len;
    const int nb = (kend + KB - 1) / KB, per = (nb + a.splits - 1) / a.splits, b0 = w.split * per, b1 = min(nb, b0 + per);
    const unsigned char* mask = d.key_mask ? d.key_mask + w.b * d.mask_batch : nullptr;
    if (d.table) {
        fill_bias(d, bias, w.head0, a.gp, tid, NT);
        __syncthreads();
    }
    const float* brow = d.table ? bias + hg * (2 * d.reach + 1) + d.reach : nullptr;
    const T* kb = reinterpret_cast<const T*>(d.k) + w.b * d.k_batch + (long long)w.kvh * d.dh;
    const T* vb = reinterpret_cast<const T*>(d.v) + w.b * d.v_batch + (long long)w.kvh * d.dh;
    u32x4 qf[NC];
    const T* qrow = reinterpret_cast<const T*>(d.q) + w.b * d.q_batch + i * d.q_row + (long long)h * d.dh;
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = row_frag_global<T, 16>(qrow, c, d.dh, ok, lane);
    const TileFrag<T, DH, 16> tf(lane);
    f32x4 o[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[mt] = zero_acc<16>();
    float m = NEG_INF, l = 0.f;
    Block x, y;
    x.copy.init(vb, d.v_row, lane);
    y.copy.init(vb, d.v_row, lane);
    const uint64_t seed = d.drop_p > 0.f ? drop_seed_value(a.seed) : 0;
    const int first = b0 + wave;
    if (first < b1) x.load(d, kb, vb, mask, first * KB, kend, va[wave], lane);
    auto block = [&](int t, Block& cur, const T* vs, Block& next, T* vn) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0x0070);                   // this block has arrived, the buffer of the one before is read
        if (t + NW < b1) next.load(d, kb, vb, mask, (t + NW) * KB, kend, vn, lane);
        f32x4 s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            s[b] = zero_acc<16>();
#pragma unroll
            for (int c = 0; c < NC; ++c) s[b] = mma<T, 16>(cur.k[b][c], qf[c], s[b]);
        }
        float mx = m;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = t * KB + 16 * b + 4 * g + e;
                float z = s[b][e] * a.sc2;
                if (brow) z += brow[min(max(j - pos, -d.reach), d.reach)];
                if (!((cur.ok[b] >> (4 * g + e)) & 1) || (d.causal && j > pos)) z = NEG_INF;
                s[b][e] = z;
                mx = fmaxf(mx, z);
            }
        mx = across_groups_max<16>(mx);
        const float base = mx == NEG_INF ? 0.f : mx, alpha = __builtin_amdgcn_exp2f(m - base);
        m = mx;
        l *= alpha;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[b][e] = __builtin_amdgcn_exp2f(s[b][e] - base);
                l += s[b][e];
                if (d.drop_p > 0.f) s[b][e] *= drop_kept(a, seed, w.b, h, i, t * KB + 16 * b + 4 * g + e);
            }
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][e] *= alpha;
        }
        const u32x4 pf = score_frag<T, 16, NB>(s, 0);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            u32x4 f;
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = cur.v[e * (DH / 64) + mt / 4][mt % 4];
            } else f = tf.cols(vs, mt * 16, 0, 0);
            o[mt] = mma<T, 16>(f, pf, o[mt]);
        }
    };
    for (int t = first; t < b1; t += 2 * NW) {
        block(t, x, va[wave], y, vb_[wave]);
        if (t + NW < b1) block(t + NW, y, vb_[wave], x, va[wave]);
    }
    // the waves' shares meet: maxima and sums first, then the outputs, each scaled by its wave
    l = across_groups_sum<16>(l);
    if (g == 0) {
        sml[wave][0][n] = m;
        sml[wave][1][n] = l;
    }
    __syncthreads();
    float M = NEG_INF, sum = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) M = fmaxf(M, sml[k][0][n]);
    const float base = M == NEG_INF ? 0.f : M;
#pragma unroll
    for (int k = 0; k < NW; ++k) sum += sml[k][1][n] * __builtin_amdgcn_exp2f(sml[k][0][n] - base);
    const float f = __builtin_amdgcn_exp2f(m - base) * (a.splits > 1 ? 1.f : sum == 0.f ? 0.f : a.inv_keep / sum);
    const long long row = ((long long)w.b * d.H + h) * d.Lq + i, total = (long long)d.B * d.H * d.Lq;
    if (ok) {
        float* p = join + (wave * rows + n) * DH;
        const int turn = n << 2;
#pragma unroll
        for (int q = 0; q < MT; ++q) {
            if constexpr (sizeof(T) == 4) {                   // q = 4 x + e: columns 64 x + 16 g + 4 e + (block 4 x + t: t)
                const int x4 = q / 4 * 4, e = q % 4;
                store4<float>(p + ((16 * x4 + 16 * g + 4 * e) ^ turn), o[x4][e] * f, o[x4 + 1][e] * f, o[x4 + 2][e] * f, o[x4 + 3][e] * f);
            } else store4<float>(p + ((16 * q + 4 * g) ^ turn), o[q][0] * f, o[q][1] * f, o[q][2] * f, o[q][3] * f);
        }
        if (wave == 0 && g == 0) {
            if (a.splits > 1) {
                a.pml[2 * (w.split * total + row)] = M;
                a.pml[2 * (w.split * total + row) + 1] = sum;
            } else if (d.lse) d.lse[row] = sum == 0.f ? POS_INF : M + __builtin_amdgcn_logf(sum);
        }
    }
    __syncthreads();
    const int vec = d.dh / 4;
    for (int k = tid; k < rows * vec; k += NT) {
        const int rr = k / vec, c = (k % vec) * 4, ri = (row0 + rr) / a.gp, rh = w.head0 + (row0 + rr) % a.gp;
        f32x4 v = *reinterpret_cast<const f32x4*>(join + rr * DH + (c ^ (rr << 2)));
#pragma unroll
        for (int q = 1; q < NW; ++q) v += *reinterpret_cast<const f32x4*>(join + (q * rows + rr) * DH + (c ^ (rr << 2)));
        if (a.splits > 1) *reinterpret_cast<f32x4*>(a.po + (w.split * total + ((long long)w.b * d.H + rh) * d.Lq + ri) * d.dh + c) = v;
        else {
            const long long at = ((long long)w.b * d.Lq + ri) * d.H * d.dh + (long long)rh * d.dh + c;
            store4<T>(reinterpret_cast<T*>(d.out) + at, v[0], v[1], v[2], v[3]);
            if (sizeof(T) == 2 && d.out32) store4<float>(d.out32 + at, v[0], v[1], v[2], v[3]);
        }
    }
}

// ---- many query rows: NW * G rows a workgroup, key tiles copied to LDS one tile ahead of the products
// Two products of 2 dh flops a pair (exp of every score between them) against K and V read once a workgroup: bound by instruction issue --
// 16 bits: the 16 exponentials and some 100 vector instructions a unit of 32 x 32 beside 16 or 8 matrix instructions --, LDS reads
// free of conflicts (64 wide vector 52 %, matrix 27 % of a busy SIMD's cycles; 128 wide causal 36 and 27, and 39 % of the wave time waiting, two
// waves a SIMD).  bf16, 8 samples x 16 heads of 64 on 4, 1021 rows x up to 2048 keys: 94 us, 500 TF; 4 x 16 heads of 128, 2048 x 2048
// causal with a bias table: 157 us, 440 TF; f32 64 x 4 heads of 256, 90 x 104: 55 us, 44 TF (one round of 256 workgroups, 64 KB of tiles each).
template <typename T, int DH, int G, int NW, int KT>
__global__ __launch_bounds__(64 * NW, G == 32 && DH * (int)sizeof(T) > 256 ? 1 : 2) void attn_tile_fwd_kernel(const AttnArgs a) {
    constexpr int NT = 64 * NW, NB = KT / G, NC = DH / (Elem<T>::epl * Blk<G>::ng), PC = KT / (Elem<T>::epl * Blk<G>::ng), MT = DH / G, nv = 4 * Blk<G>::nq;
    __shared__ __attribute__((aligned(16))) T k0[KT * DH], k1[KT * DH], v0[KT * DH], v1[KT * DH];
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* bias = reinterpret_cast<float*>(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const RowWork w(a);
    const ekaid_attn_t& d = a.d;
    const int row0 = (w.tile * NW + wave) * G, h = w.head0;
    const bool ok = row0 + lane % G < d.Lq, live = row0 < d.Lq;
    const int i = min(row0 + lane % G, d.Lq - 1), p0 = query_pos(d, w.b), pos = p0 + i, pmin = p0 + min(row0, d.Lq - 1), pmax = p0 + min(row0 + G, d.Lq) - 1;
    const int len = key_len(d, w.b), kend = d.causal ? max(0, min(len, p0 + min(d.Lq, (w.tile + 1) * NW * G))) : len;
    const int nt = (kend + KT - 1) / KT, per = (nt + a.splits - 1) / a.splits, t0 = w.split * per, t1 = min(nt, t0 + per);
    const int width = d.table ? 2 * (d.reach + BIAS_PAD) + 1 : 0;
    if (d.table) {
        fill_bias_range(d, bias, h, t0 * KT - p0 - min(d.Lq, (w.tile + 1) * NW * G) + 1, t1 * KT - p0 - w.tile * NW * G, tid, NT);
        __syncthreads();
    }
    MaskRing<KT> ring;
    ring.init(d.key_mask ? d.key_mask + w.b * d.mask_batch : nullptr, reinterpret_cast<unsigned char*>(bias + width), len, t0, tid);

    u32x4 qf[NC];
    const T* qrow = reinterpret_cast<const T*>(d.q) + w.b * d.q_batch + i * d.q_row + (long long)h * d.dh;
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = row_frag_global<T, G>(qrow, c, d.dh, ok, lane);
    TileFrag<T, DH, G> tf(lane);
    TileCopy<T, DH, KT, NW> ck, cv;
    ck.init(reinterpret_cast<const T*>(d.k) + w.b * d.k_batch + (long long)w.kvh * d.dh, d.k_row, lane);
    cv.init(reinterpret_cast<const T*>(d.v) + w.b * d.v_batch + (long long)w.kvh * d.dh, d.v_row, lane);
    typename Blk<G>::acc o[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[mt] = zero_acc<G>();
    float m = NEG_INF, l = 0.f;
    if (t0 < t1) {
        ck.issue(k0, t0 * KT, kend, d.dh, ring.tile(t0), wave);
        cv.issue(v0, t0 * KT, kend, d.dh, ring.tile(t0), wave);
    }
    auto tile = [&](int t, const T* ks, const T* vs, T* kn, T* vn) __attribute__((always_inline)) {
        settle();
        ring.step(t);
        if (t + 1 < t1) {
            ck.issue(kn, (t + 1) * KT, kend, d.dh, ring.tile(t + 1), wave);
            cv.issue(vn, (t + 1) * KT, kend, d.dh, ring.tile(t + 1), wave);
        }
        if (!live || (d.causal && t * KT > pmax)) return;
        if constexpr (DH * sizeof(T) > 128) tf.refresh();
        typename Blk<G>::acc s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b] = zero_acc<G>();
        fragment_loop<T, G, NC * NB>([&](int n) __attribute__((always_inline)) { return tf.rows(ks, (n % NB) * G, n / NB); },
                                  [&](int n, u32x4 x) __attribute__((always_inline)) { s[n % NB] = mma<T, G>(x, qf[n / NB], s[n % NB]); });
        const Affine f = scores_by_row<G, NB>(a, s, t * KT, len, pos, pmin, pmax, d.table ? bias : nullptr, ring.tile(t), lane);
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < nv; ++r) mx = fmaxf(mx, s[b][r]);
        const float mn = across_groups_max<G>(mx) * f.mult + f.add;                // (mult >= 0)
        if (__any(mn > m + 6.f)) {                        // m need not be the maximum, only near it: powers up to 2^6 lose nothing, and most
            const float up = fmaxf(m, mn), alpha = __builtin_amdgcn_exp2f(m - (up == NEG_INF ? 0.f : up));      // tiles leave the outputs alone
            m = up;
            l *= alpha;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < nv; ++e) o[mt][e] *= alpha;
        }
        const float shift = f.add - (m == NEG_INF ? 0.f : m);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < nv; ++r) {
                s[b][r] = __builtin_amdgcn_exp2f(s[b][r] * f.mult + shift);
                l += s[b][r];
            }
        if (d.drop_p > 0.f) drop_scores<G, NB>(a, s, w.b, h, i, t * KT, lane);
        u32x4 pf[PC];
#pragma unroll
        for (int c = 0; c < PC; ++c) pf[c] = score_frag<T, G, NB>(s, c);
        fragment_loop<T, G, PC * MT>([&](int n) __attribute__((always_inline)) { return tf.cols(vs, (n % MT) * G, 0, n / MT); },
                                  [&](int n, u32x4 x) __attribute__((always_inline)) { o[n % MT] = mma<T, G>(x, pf[n / MT], o[n % MT]); });
    };
    for (int t = t0; t < t1; t += 2) {
        tile(t, k0, v0, k1, v1);
        if (t + 1 < t1) tile(t + 1, k1, v1, k0, v0);
    }
    write_rows<T, DH, G>(a, w, o, m, l, i, h, ok, lane);
}

// joins the partial outputs of a split launch: one wave per row
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a) {
    const ekaid_attn_t& d = a.d;
    const long long rows = (long long)d.B * d.H * d.Lq, row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows) return;
    float m = NEG_INF;
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.pml[2 * (s * rows + row)]);
    m = wave_max(m);
    const float base = m == NEG_INF ? 0.f : m;
    float l = 0.f;
    for (int s = lane; s < a.splits; s += 64) l += a.pml[2 * (s * rows + row) + 1] * __builtin_amdgcn_exp2f(a.pml[2 * (s * rows + row)] - base);
    l = wave_sum(l);
    const float inv = l == 0.f ? 0.f : a.inv_keep / l;
    const long long i = row % d.Lq, bh = row / d.Lq;
    T* out = reinterpret_cast<T*>(d.out) + ((bh / d.H) * d.Lq + i) * d.H * d.dh + (bh % d.H) * d.dh;
    for (int c = 4 * lane; c < d.dh; c += 256) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < a.splits; ++s) {
            const float f = __builtin_amdgcn_exp2f(a.pml[2 * (s * rows + row)] - base);
            const f32x4 v = *reinterpret_cast<const f32x4*>(a.po + (s * rows + row) * d.dh + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += f * v[e];
        }
        acc *= inv;
        store4<T>(out + c, acc[0], acc[1], acc[2], acc[3]);
        if (sizeof(T) == 2 && d.out32) store4<float>(d.out32 + (out - reinterpret_cast<T*>(d.out)) + c, acc[0], acc[1], acc[2], acc[3]);
    }
    if (lane == 0 && d.lse) d.lse[row] = l == 0.f ? POS_INF : m + __builtin_amdgcn_logf(l);
}

// ---- host side
int attn_lds_limit(const void* fn, int bytes) {
    if (func_attr_once(fn) && hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
        (void)hipGetLastError();
        set_error("attention: cannot raise the LDS limit");
        return EKAID_ERR_LAUNCH;
    }
    return EKAID_OK;
}

int attn_check(const ekaid_attn_t* a, const char* who) {
    if (!a) { set_error("%s: null descriptor", who); return EKAID_ERR_ARG; }
    if (a->dtype < EKAID_F32 || a->dtype > EKAID_F16) { set_error("%s: dtype %d", who, a->dtype); return EKAID_ERR_ARG; }
    if (a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->H < 1 || a->KV < 1 || a->H % a->KV) {
        set_error("%s: bad sizes B=%d Lq=%d Lk=%d H=%d KV=%d", who, a->B, a->Lq, a->Lk, a->H, a->KV);
        return EKAID_ERR_ARG;
    }
    if (a->dh < 8 || a->dh > 256 || a->dh % 8) { set_error("%s: head width %d (a multiple of 8 up to 256)", who, a->dh); return EKAID_ERR_UNSUPPORTED; }
    const int esz = a->dtype == EKAID_F32 ? 4 : 2, epl = 16 / esz;
    if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v) & 15) { set_error("%s: operands must be 16-byte aligned", who); return EKAID_ERR_ARG; }
    const long long st[6] = {a->q_batch, a->q_row, a->k_batch, a->k_row, a->v_batch, a->v_row};
    for (long long s : st)
        if (s < 0 || s % epl) { set_error("%s: stride %lld is not a whole number of 16-byte vectors", who, s); return EKAID_ERR_ARG; }
    if (!(a->drop_p >= 0.f && a->drop_p < 1.f)) { set_error("%s: dropout probability %g", who, (double)a->drop_p); return EKAID_ERR_ARG; }
    if (a->table) {
        if (a->table_dtype < EKAID_F32 || a->table_dtype > EKAID_F16 || a->n_border < 0 || a->n_border >= ATTN_MAX_BUCKETS || a->reach < 1 ||
            a->reach > EKAID_ATTN_MAX_REACH || (a->n_border && a->border[a->n_border - 1] > a->reach)) {
            set_error("%s: relative bias: table_dtype=%d n_border=%d reach=%d", who, a->table_dtype, a->n_border, a->reach);
            return EKAID_ERR_ARG;
        }
        for (int i = 0; i < a->n_border; ++i)
            if (a->border[i] < (i ? a->border[i - 1] : 1)) { set_error("%s: borders must not descend, from 1 on", who); return EKAID_ERR_ARG; }
    }
    // a launch counts its threads in 32 bits: 256 a head of up to 16 rows, four a row or key, 64 a table entry
    const long long bh = (long long)a->B * a->H;
    if (bh >= (1 << 24) || bh * ((long long)std::max(a->Lq, a->Lk) + 128) >= (1ll << 30) || (a->table && a->H >= (1 << 18))) {
        set_error("%s: too many rows for one launch", who);
        return EKAID_ERR_UNSUPPORTED;
    }
    return EKAID_OK;
}

struct FwdPlan { int few, g, nw, gp, tiles, splits; size_t ws; };

// Waves of 16 rows a workgroup: as few rows as possible beyond R (a wave on rows that do not exist costs as much as one on rows that do),
// weighed with what smaller workgroups cost: tiles copied more often; with 64 KB of tiles (`wide`: 256-wide f32 heads) also fewer waves on
// a compute unit, whose LDS holds two workgroups (64 x 4 heads x 90 x 104: 55 us forward with 4 waves, 82 with 2)
int waves_for_rows(int R, bool wide) {
    int best = 4, cost = 1 << 30;
    for (int nw = 4; nw >= 1; nw >>= 1) {
        const int c = cdiv(R, 16 * nw) * 16 * nw * (nw == 4 ? 8 : nw == 2 ? (wide ? 14 : 9) : wide ? 24 : 12);
        if (c < cost) { cost = c; best = nw; }
    }
    return best;
}

static FwdPlan fwd_plan(const ekaid_attn_t* a) {
    FwdPlan p;
    const int group = a->H / a->KV, esz = a->dtype == EKAID_F32 ? 4 : 2;
    // up to 16 query rows a head: the kernel whose waves split the keys; the heads that share keys go into its rows while those fit twice
    p.few = a->Lq <= 16;
    p.gp = p.few && a->Lq * group <= 32 && (!a->table || group * (2 * a->reach + 1) <= 7900) ? group : 1;
    int per_tile, keys;
    if (p.few) {
        p.g = 16;
        p.nw = 4;
        per_tile = 16;
        keys = 4 * (esz == 4 ? 16 : 32);
    } else {
        p.g = a->Lq <= 64 || (esz == 4 && a->dh > 128) ? 16 : 32;
        p.nw = p.g == 32 ? 4 : waves_for_rows(a->Lq, esz == 4 && a->dh > 128);
        per_tile = p.g * p.nw;
        keys = attn_kt(esz, a->dh, p.g);
    }
    p.tiles = cdiv(a->Lq * p.gp, per_tile);
    const long long wgs = (long long)a->B * (a->H / p.gp) * p.tiles;
    const int steps = cdiv(a->Lk, keys);
    long long s = 1;
    const long long want = 4 * 512 / p.nw;
    if (wgs < want / 2 && steps > 1) s = (want + wgs - 1) / (wgs > 0 ? wgs : 1);
    if (s > (steps + 1) / 2) s = (steps + 1) / 2;
    p.splits = (int)(s < 1 ? 1 : s);
    p.ws = p.splits > 1 ? (size_t)p.splits * a->B * a->H * a->Lq * (a->dh + 2) * sizeof(float) : 0;
    return p;
}

template <typename T, int DH> static int launch_few(const AttnArgs& a, int grid, hipStream_t st) {
    const int rows = std::min(16, a.d.Lq * a.gp);
    const size_t lds = (sizeof(T) == 4 ? (size_t)4 * rows * DH * 4 : 0) + (a.d.table ? (size_t)a.gp * (2 * a.d.reach + 1) * 4 : 0);
    if (int rc = attn_lds_limit((const void*)attn_few_kernel<T, DH, 4>, sizeof(T) == 4 ? 100 * 1024 : 32 * 1024 - 1024)) return rc;
    hipLaunchKernelGGL((attn_few_kernel<T, DH, 4>), dim3(grid), dim3(256), lds, st, a);
    return check_launch("attn_fwd");
}
template <typename T, int DH, int G, int NW> static int launch_tile(const AttnArgs& a, int grid, hipStream_t st) {
    constexpr int KT = attn_kt((int)sizeof(T), DH, G);
    const size_t lds = (a.d.table ? (size_t)(2 * (a.d.reach + BIAS_PAD) + 1) * 4 : 0) + 4 * KT;
    if (int rc = attn_lds_limit((const void*)attn_tile_fwd_kernel<T, DH, G, NW, KT>, 96 * 1024)) return rc;
    hipLaunchKernelGGL((attn_tile_fwd_kernel<T, DH, G, NW, KT>), dim3(grid), dim3(64 * NW), lds, st, a);
    return check_launch("attn_fwd");
}
template <typename T, int DH> static int pick_fwd(const AttnArgs& a, const FwdPlan& p, int grid, hipStream_t st) {
    if (p.few) return launch_few<T, DH>(a, grid, st);
    if constexpr (!(sizeof(T) == 4 && DH > 128))
        if (p.g == 32) return launch_tile<T, DH, 32, 4>(a, grid, st);
    if (p.nw == 1) return launch_tile<T, DH, 16, 1>(a, grid, st);
    if (p.nw == 2) return launch_tile<T, DH, 16, 2>(a, grid, st);
    return launch_tile<T, DH, 16, 4>(a, grid, st);
}
template <typename T> static int run_fwd(const AttnArgs& a, const FwdPlan& p, hipStream_t st) {
    const int grid = a.d.B * (a.d.H / p.gp) * p.tiles * p.splits;
    const int rc = a.d.dh <= 64 ? pick_fwd<T, 64>(a, p, grid, st) : a.d.dh <= 128 ? pick_fwd<T, 128>(a, p, grid, st) : pick_fwd<T, 256>(a, p, grid, st);
    if (rc || p.splits == 1) return rc;
    hipLaunchKernelGGL(attn_join_kernel<T>, dim3(cdiv((long long)a.d.B * a.d.H * a.d.Lq, 4)), dim3(256), 0, st, a);
    return check_launch("attn_join");
}
}  // namespace ekaid

extern "C" size_t ekaid_attn_workspace_bytes(const ekaid_attn_t* a, int backward) {
    using namespace ekaid;
    if (attn_check(a, "attn_workspace_bytes") || a->B == 0 || a->Lq == 0) return 0;
    return backward ? attn_bwd_workspace(a) : fwd_plan(a).ws;
}

extern "C" int ekaid_attn_fwd(const ekaid_attn_t* a, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace ekaid;
    if (int rc = attn_check(a, "attn_fwd")) return rc;
    if (a->B == 0 || a->Lq == 0) return EKAID_OK;
    if (!a->q || !a->out || (a->Lk && (!a->k || !a->v))) { set_error("attn_fwd: null operand"); return EKAID_ERR_ARG; }
    const FwdPlan p = fwd_plan(a);
    if (workspace_bytes < p.ws || (p.ws && !workspace)) { set_error("attn_fwd: workspace of %zu bytes needed", p.ws); return EKAID_ERR_ARG; }
    AttnArgs k = {};
    k.d = *a;
    k.seed = DS(a->drop_seed);
    k.inv_keep = 1.f / (1.f - a->drop_p);
    k.sc2 = a->scale * LOG2E;
    k.gp = p.gp;
    k.near = !p.few || a->Lk > 512 ? 1 : a->KV % 4 == 0 ? 4 : a->KV % 2 == 0 ? 2 : 1;
    k.tiles = p.tiles;
    k.splits = p.splits;
    k.po = (float*)workspace;
    k.pml = k.po + (size_t)p.splits * a->B * a->H * a->Lq * a->dh;
    hipStream_t st = (hipStream_t)stream;
    return a->dtype == EKAID_F32 ? run_fwd<float>(k, p, st) : a->dtype == EKAID_BF16 ? run_fwd<__bf16>(k, p, st) : run_fwd<_Float16>(k, p, st);
}
