// Backward of the attention operators (include/ekaid_hip.h: ekaid_attn_t).  Scores are formed again from q, k and the stored log2
// denominators; two kernels, so that no output is an atomic target: dq with one workgroup per block of query rows, dk / dv (and the bias
// table's sums) with one per block of keys, walking the rows of every head that shares them.  Seven products where the formula has five.
#include "attn.h"
#include <algorithm>

namespace ekaid {

// f16 only: powers of two that keep the score gradients P (keep dP - delta) inside the f16 range whatever the scale of the incoming gradient
// (a loss divided by thousands of tokens) and of the values: |dP_ij| <= |dout_i| |v_j| and |delta_i| <= inv_keep |dout_i| max |v|, so their
// difference is at most 2 inv_keep |dout_i| max |v|, which is brought to [2^13, 2^15).  Exact, taken out in f32.
template <typename T> __device__ __forceinline__ float ds_scale(const AttnArgs& a, float dout2, float v2) {
    if constexpr (__is_same(T, _Float16)) {
        const float n = dout2 * v2;                           // (f16 rows: within 2^-96 .. 2^81)
        if (!(n > 0.f) || n == POS_INF) return 1.f;
        const int e = (int)((__builtin_bit_cast(uint32_t, n) >> 23) & 255) - 127;          // n in [2^e, 2^(e+1))
        return ldexpf(1.f, 13 - (e >> 1) - a.keep_exp);
    } else return 1.f;
}
// largest squared norm of the value rows a sample's rows may attend, by parts of the keys; one workgroup a part.  Reads the values once more:
// 8 samples x 4 heads of 64, up to 2048 keys 5.1 us; 4 x 16 heads of 128, 2048 keys (34 MB) 9.1 us, of 346 and 680 us of whole passes
__global__ __launch_bounds__(256) void attn_vnorm_kernel(const AttnArgs a) {
    const ekaid_attn_t& d = a.d;
    const int part = blockIdx.x % a.v_parts, bk = blockIdx.x / a.v_parts, b = bk % d.B, kvh = bk / d.B, tid = threadIdx.x;
    const int len = key_len(d, b), p0 = query_pos(d, b), per = (d.Lk + a.v_parts - 1) / a.v_parts;
    int lanes = 1;                                            // that share a row, 16 bytes each
    while (8 * lanes < d.dh) lanes <<= 1;
    const int col = tid % lanes * 8, step = 256 / lanes, end = min(len, (part + 1) * per);
    const unsigned char* mask = d.key_mask ? d.key_mask + b * d.mask_batch : nullptr;
    const _Float16* v = reinterpret_cast<const _Float16*>(d.v) + b * d.v_batch + (long long)kvh * d.dh + col;
    float mx = 0.f;
    for (int j0 = part * per; j0 < end; j0 += step) {         // (whole waves stay together for the exchange)
        const int j = j0 + tid / lanes;
        float s = 0.f;
        if (j < end && col < d.dh && (!d.causal || j - d.Lq < p0) && (!mask || mask[j])) {
            const f16x8 x = *reinterpret_cast<const f16x8*>(v + j * d.v_row);
#pragma unroll
            for (int e = 0; e < 8; ++e) s += (float)x[e] * (float)x[e];
        }
        for (int o = 1; o < lanes; o <<= 1) s += __shfl_xor(s, o, 64);
        mx = fmaxf(mx, s);
    }
    __shared__ float part_max[4];
    mx = wave_max(mx);
    if ((tid & 63) == 0) part_max[tid >> 6] = mx;
    __syncthreads();
    if (tid == 0) a.vn[(long long)(b * d.KV + kvh) * a.v_parts + part] = fmaxf(fmaxf(part_max[0], part_max[1]), fmaxf(part_max[2], part_max[3]));
}
// the largest of them for one key head, in every lane
template <typename T> __device__ __forceinline__ float value_norm2(const AttnArgs& a, int b, int kvh, int lane) {
    if constexpr (!__is_same(T, _Float16)) return 0.f;
    float mx = 0.f;
    const float* n = a.vn + (long long)(b * a.d.KV + kvh) * a.v_parts;
    for (int x = lane; x < a.v_parts; x += 64) mx = fmaxf(mx, n[x]);
    return wave_max(mx);
}

// dq: lane = query row.  Units of 32 keys of a tile: scores and dP of a unit, then its share of dq.  Three products a pair; bound as the
// forward.  bf16, 8 samples x 16 heads of 64 on 4, 1021 rows x up to 2048 keys: 114 us, 625 TF; 4 x 16 heads of 128, 2048 x 2048 causal with a
// bias table: 209 us, 490 TF.
// With a bias table the kernel also sums every row's score gradients: with delta = sum_j P dP they would be zero, so what they are is the
// error of <dout, out> against it (out was formed from probabilities rounded to the type).  Added to delta, it makes the score gradients of
// dk / dv and the table's long sums exact to f32.
template <typename T, int DH, int G, int NW, int KT, bool REL>
__global__ __launch_bounds__(64 * NW, G == 32 && DH * (int)sizeof(T) > 256 ? 1 : 2) void attn_dq_kernel(const AttnArgs a) {
    constexpr int NT = 64 * NW, U = KT < 32 ? KT : 32, NB = U / G, NC = DH / (Elem<T>::epl * Blk<G>::ng), PC = U / (Elem<T>::epl * Blk<G>::ng), MT = DH / G;
    constexpr int nq = Blk<G>::nq, ng = Blk<G>::ng, nv = 4 * nq;
    __shared__ __attribute__((aligned(16))) T k0[KT * DH], k1[KT * DH], v0[KT * DH], v1[KT * DH];
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane / G, width = REL ? 2 * (a.d.reach + BIAS_PAD) + 1 : 0;
    float* red = reinterpret_cast<float*>(smem);              // [NW] row-norm maxima
    float* bias = red + NW;                                   // padded table of the head
    unsigned char* kms = reinterpret_cast<unsigned char*>(bias + width);
    const RowWork w(a);
    const ekaid_attn_t& d = a.d;
    const int h = w.head0, row0 = (w.tile * NW + wave) * G;
    const bool ok = row0 + lane % G < d.Lq, live = row0 < d.Lq;
    const int i = min(row0 + lane % G, d.Lq - 1), p0 = query_pos(d, w.b), pos = p0 + i, pmin = p0 + min(row0, d.Lq - 1), pmax = p0 + min(row0 + G, d.Lq) - 1;
    const int len = key_len(d, w.b), kend = d.causal ? max(0, min(len, p0 + min(d.Lq, (w.tile + 1) * NW * G))) : len;
    const int nt = (kend + KT - 1) / KT, per = (nt + a.splits - 1) / a.splits, t0 = w.split * per, t1 = min(nt, t0 + per);
    if constexpr (REL) {
        fill_bias_range(d, bias, h, t0 * KT - p0 - min(d.Lq, (w.tile + 1) * NW * G) + 1, t1 * KT - p0 - w.tile * NW * G, tid, NT);
        __syncthreads();
    }
    MaskRing<KT> ring;
    ring.init(d.key_mask ? d.key_mask + w.b * d.mask_batch : nullptr, kms, len, t0, tid);

    TileFrag<T, DH, G> tf(lane);
    TileCopy<T, DH, KT, NW> ck, cv;
    ck.init(reinterpret_cast<const T*>(d.k) + w.b * d.k_batch + (long long)w.kvh * d.dh, d.k_row, lane);
    cv.init(reinterpret_cast<const T*>(d.v) + w.b * d.v_batch + (long long)w.kvh * d.dh, d.v_row, lane);
    u32x4 qf[NC], gf[NC];
    const long long orow = ((long long)w.b * d.Lq + i) * d.H * d.dh + (long long)h * d.dh;
    const T* qrow = reinterpret_cast<const T*>(d.q) + w.b * d.q_batch + i * d.q_row + (long long)h * d.dh;
    const T* grow = reinterpret_cast<const T*>(d.dout) + orow;
    const T* yrow = reinterpret_cast<const T*>(d.out) + orow;
    float delta = 0.f, n2 = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        qf[c] = row_frag_global<T, G>(qrow, c, d.dh, ok, lane);
        gf[c] = row_frag_global<T, G>(grow, c, d.dh, ok, lane);
        if (sizeof(T) == 2 && d.out32) {
            const int col = (c * ng + g) * Elem<T>::epl;
            f32x4 y0 = {0.f, 0.f, 0.f, 0.f}, y1 = y0;
            if (ok && col < d.dh) {
                y0 = *reinterpret_cast<const f32x4*>(d.out32 + orow + col);
                y1 = *reinterpret_cast<const f32x4*>(d.out32 + orow + col + 4);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) delta += elem<T>(gf[c], e) * y0[e] + elem<T>(gf[c], (4 + e) % Elem<T>::epl) * y1[e];
        } else {
            const u32x4 y = row_frag_global<T, G>(yrow, c, d.dh, ok, lane);
#pragma unroll
            for (int e = 0; e < Elem<T>::epl; ++e) delta += elem<T>(gf[c], e) * elem<T>(y, e);
        }
#pragma unroll
        for (int e = 0; e < Elem<T>::epl; ++e) n2 += elem<T>(gf[c], e) * elem<T>(gf[c], e);
    }
    if (t0 < t1) {
        ck.issue(k0, t0 * KT, kend, d.dh, ring.tile(t0), wave);
        cv.issue(v0, t0 * KT, kend, d.dh, ring.tile(t0), wave);
    }
    delta = across_groups_sum<G>(delta);
    n2 = across_groups_sum<G>(n2);
    const long long srow = ((long long)w.b * d.H + h) * d.Lq + i;
    const float lse = ok ? d.lse[srow] : POS_INF;
    const bool empty = lse == POS_INF;                        // a row without any key: zeros, whatever dout holds there
    if (empty) delta = 0.f;
    if (ok && g == 0 && w.split == 0 && (!REL || a.splits > 1)) a.delta[srow] = delta;
    const float rs = ds_scale<T>(a, n2, value_norm2<T>(a, w.b, w.kvh, lane));
    if constexpr (__is_same(T, _Float16)) {
        const float mx = wave_max(n2);
        if (lane == 0) red[wave] = mx;
    }
    typename Blk<G>::acc o[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[mt] = zero_acc<G>();
    float rowsum = 0.f;
    const uint64_t seed = d.drop_p > 0.f ? drop_seed_value(a.seed) : 0;

    auto unit = [&](int j0, const T* ks, const T* vs, int r0, const unsigned char* km) __attribute__((always_inline)) {
        if constexpr (DH * sizeof(T) > 128) tf.refresh();
        typename Blk<G>::acc s[NB], dp[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            s[b] = zero_acc<G>();
            dp[b] = zero_acc<G>();
        }
        fragment_loop<T, G, NC * NB * 2>([&](int n) __attribute__((always_inline)) { return tf.rows(n & 1 ? vs : ks, r0 + (n / 2 % NB) * G, n / 2 / NB); },
                                      [&](int n, u32x4 x) __attribute__((always_inline)) {
                                          const int b = n / 2 % NB, c = n / 2 / NB;
                                          if (n & 1) dp[b] = mma<T, G>(x, gf[c], dp[b]);
                                          else s[b] = mma<T, G>(x, qf[c], s[b]);
                                      });
        const Affine f = scores_by_row<G, NB>(a, s, j0, len, pos, pmin, pmax, REL ? bias : nullptr, km, lane);
        const float shift = f.add - lse;
        if (d.drop_p > 0.f) {
#pragma unroll
            for (int q = 0; q < NB * nq; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) dp[q / nq][4 * (q % nq) + e] *= drop_keep(a, seed, w.b, h, i, j0 + 4 * ng * q + 4 * g + e);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < nv; ++r) s[b][r] = __builtin_amdgcn_exp2f(s[b][r] * f.mult + shift) * (dp[b][r] - delta);
        if constexpr (REL) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < nv; ++r) rowsum += s[b][r];
        }
        if constexpr (__is_same(T, _Float16)) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < nv; ++r) s[b][r] *= rs;
        }
        u32x4 sf[PC];
#pragma unroll
        for (int c = 0; c < PC; ++c) sf[c] = score_frag<T, G, NB>(s, c);
        fragment_loop<T, G, PC * MT>([&](int n) __attribute__((always_inline)) { return tf.cols(ks, (n % MT) * G, r0, n / MT); },
                                  [&](int n, u32x4 x) __attribute__((always_inline)) { o[n % MT] = mma<T, G>(x, sf[n / MT], o[n % MT]); });
    };
    auto tile = [&](int t, const T* ks, const T* vs, T* kn, T* vn) __attribute__((always_inline)) {
        settle();
        ring.step(t);
        if (t + 1 < t1) {
            ck.issue(kn, (t + 1) * KT, kend, d.dh, ring.tile(t + 1), wave);
            cv.issue(vn, (t + 1) * KT, kend, d.dh, ring.tile(t + 1), wave);
        }
        const unsigned char* km = ring.tile(t);
#pragma unroll
        for (int u = 0; u < KT / U; ++u) {
            const int j0 = t * KT + u * U;
            if (live && j0 < kend && !(d.causal && j0 > pmax)) unit(j0, ks, vs, u * U, km ? km + u * U : nullptr);
        }
    };
    for (int t = t0; t < t1; t += 2) {
        tile(t, k0, v0, k1, v1);
        if (t + 1 < t1) tile(t + 1, k1, v1, k0, v0);
    }
    if constexpr (REL) {
        rowsum = empty ? 0.f : across_groups_sum<G>(rowsum);
        if (ok && g == 0) {
            if (a.splits > 1) a.eps[(long long)w.split * d.B * d.H * d.Lq + srow] = rowsum;
            else a.delta[srow] = delta + rowsum;
        }
    }
    if constexpr (__is_same(T, _Float16)) {
        __syncthreads();
        if (tid == 0) {
            float mx = red[0];
            for (int x = 1; x < NW; ++x) mx = fmaxf(mx, red[x]);
            a.nrm[(long long)(w.b * d.H + h) * a.dq_parts + w.tile * a.splits + w.split] = mx;
        }
    }
    if (!ok) return;
    const float f = d.scale / rs;
    float* part = a.po + w.split * ((long long)d.B * d.Lq * d.H * d.dh) + orow;
    T* out = reinterpret_cast<T*>(d.dq) + orow;
#pragma unroll
    for (int q = 0; q < MT * nq; ++q) {
        const int col = 4 * ng * q + 4 * g, r = 4 * (q % nq);
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = empty ? 0.f : o[q / nq][r + e] * f;
        if (col >= d.dh) continue;
        if (a.splits > 1) store4<float>(part + col, x[0], x[1], x[2], x[3]);
        else store4<T>(out + col, x[0], x[1], x[2], x[3]);
    }
}

// dk, dv: lane = key; the rows of every head that shares it go by in tiles, in units of 32.  What a lane without a valid key computes stays in
// that lane and is replaced by zero at the end.  Four products a pair.  The same shapes as at dq: 159 us, 600 TF, and 335 us, 410 TF.
// 64 wide no unit is full (vector 38 %, matrix 35 %, LDS 26 % of a busy compute unit's cycles): one round of 512 workgroups, two a compute
// unit and two waves a SIMD, near a third of them on keys behind their sample's length.  128 wide a block of 32 keys would leave one wave a
// SIMD its registers, so blocks of 16 read LDS twice as often; 41 % of the wave time is waiting (vector 31 %, matrix 20 %, LDS 26 %).  The
// table's sums, met by the 15 % of the pairs within the reach, cost it their LDS, registers and fences: 275 us without a table.
template <typename T, int DH, int G, int NW, int QT, bool REL>
__global__ __launch_bounds__(64 * NW, DH * (int)sizeof(T) * G > 4096 ? 1 : G == 16 && sizeof(T) == 2 && !(REL && DH > 64) ? 3 : 2) void attn_dkv_kernel(const AttnArgs a) {
    constexpr int NT = 64 * NW, U = QT < 32 ? QT : 32, NB = U / G, NC = DH / (Elem<T>::epl * Blk<G>::ng), PC = U / (Elem<T>::epl * Blk<G>::ng), MT = DH / G;
    constexpr int nq = Blk<G>::nq, ng = Blk<G>::ng;
    __shared__ __attribute__((aligned(16))) T q0s[QT * DH], q1s[QT * DH], g0s[QT * DH], g1s[QT * DH];
    __shared__ __attribute__((aligned(16))) float l0s[QT], l1s[QT], d0s[QT], d1s[QT];      // log2 denominators, deltas
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane / G, width = REL ? 2 * a.d.reach + 1 : 0;
    float* bias = reinterpret_cast<float*>(smem);             // padded table of the head
    float* dsum = bias + (REL ? width + 2 * BIAS_PAD : 0);    // [NW][width]: this wave's sums of score gradients by distance
    float* far = dsum + NW * width;                           // [NW][2]
    constexpr int DIAG = U + G - 1, DP = U + 4;               // diagonals of a unit; places of a diagonal (one a row)
    float* skew = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(far + 2 * NW) + 15) & ~(uintptr_t)15) + wave * DIAG * DP;      // [NW][DIAG][DP]
    const ekaid_attn_t& d = a.d;
    const int wi = die_order(blockIdx.x, gridDim.x), tl = wi % a.tiles, split = (wi / a.tiles) % a.splits, bk = wi / a.tiles / a.splits;
    const int b = bk % d.B, kvh = bk / d.B, group = d.H / d.KV;
    const int len = key_len(d, b), p0 = query_pos(d, b), j0 = tl * NW * G, jw = j0 + wave * G, j = jw + lane % G;
    const unsigned char* mask = d.key_mask ? d.key_mask + b * d.mask_batch : nullptr;
    const int kend = d.causal ? max(0, min(len, p0 + d.Lq)) : len;                                        // keys that some row may attend
    const bool ok = j < kend && (!mask || mask[j]), live = jw < len;
    const int qtiles = (d.Lq + QT - 1) / QT, first = d.causal ? min(qtiles, max(0, j0 - p0) / QT) : 0, run = qtiles - first;
    const int items = j0 < len ? group * run : 0, per = (items + a.splits - 1) / a.splits, t0 = split * per, t1 = min(items, t0 + per);

    u32x4 kf[NC], vf[NC];
    const int jr = ok ? j : 0;
    const T* krow = reinterpret_cast<const T*>(d.k) + b * d.k_batch + jr * d.k_row + (long long)kvh * d.dh;
    const T* vrow = reinterpret_cast<const T*>(d.v) + b * d.v_batch + jr * d.v_row + (long long)kvh * d.dh;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        kf[c] = row_frag_global<T, G>(krow, c, d.dh, ok, lane);
        vf[c] = row_frag_global<T, G>(vrow, c, d.dh, ok, lane);
    }
    // f16: probabilities enter dv's product times 2^(15 - keep_exp) (kept ones at most 2^15): one in 2^14 keys or more would be below f16's
    // normal range.  Exact, taken out in f32.
    const float ps = __is_same(T, _Float16) ? ldexpf(1.f, 15 - a.keep_exp) : 1.f;
    float rs = 1.f;
    if constexpr (__is_same(T, _Float16)) {                   // the largest |dout| row of the heads that share these keys
        float mx = 0.f;
        const float* n = a.nrm + (long long)(b * d.H + kvh * group) * a.dq_parts;
        for (int x = lane; x < group * a.dq_parts; x += 64) mx = fmaxf(mx, n[x]);
        rs = ds_scale<T>(a, wave_max(mx), value_norm2<T>(a, b, kvh, lane));
    }
    typename Blk<G>::acc dk[MT], dv[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        dk[mt] = zero_acc<G>();
        dv[mt] = zero_acc<G>();
    }
    TileFrag<T, DH, G> tf(lane);
    TileCopy<T, DH, QT, NW> cq, cg;
    auto fetch = [&](int t, T* qs, T* gs, float* ls, float* ds) __attribute__((always_inline)) {
        const int h = kvh * group + t / run, r0 = (first + t % run) * QT;
        cq.init(reinterpret_cast<const T*>(d.q) + b * d.q_batch + (long long)h * d.dh, d.q_row, lane);
        cg.init(reinterpret_cast<const T*>(d.dout) + (long long)b * d.Lq * d.H * d.dh + (long long)h * d.dh, (long long)d.H * d.dh, lane);
        cq.issue(qs, r0, d.Lq, d.dh, nullptr, wave);
        cg.issue(gs, r0, d.Lq, d.dh, nullptr, wave);
        const long long row = ((long long)b * d.H + h) * d.Lq + min(r0 + lane, d.Lq - 1);
        if (lane < QT) {
            if (wave == 0) __builtin_amdgcn_global_load_lds((global_void)(d.lse + row), (lds_void)ls, 4, 0, 0);
            if (wave == NW - 1) __builtin_amdgcn_global_load_lds((global_void)(a.delta + row), (lds_void)ds, 4, 0, 0);
        }
    };
    float far_back = 0.f, far_ahead = 0.f;
    const uint64_t seed = d.drop_p > 0.f ? drop_seed_value(a.seed) : 0;
    // rows i0 .. i0 + U of head h, at tile row r0
    auto unit = [&](int h, int i0, int r0, const T* qs, const T* gs, const float* ls, const float* ds) __attribute__((always_inline)) {
        if constexpr (DH * sizeof(T) > 128) tf.refresh();
        typename Blk<G>::acc s[NB], dp[NB];
#pragma unroll
        for (int x = 0; x < NB; ++x) {
            s[x] = zero_acc<G>();
            dp[x] = zero_acc<G>();
        }
        fragment_loop<T, G, NC * NB * 2>([&](int n) __attribute__((always_inline)) { return tf.rows(n & 1 ? gs : qs, r0 + (n / 2 % NB) * G, n / 2 / NB); },
                                      [&](int n, u32x4 x) __attribute__((always_inline)) {
                                          const int y = n / 2 % NB, c = n / 2 / NB;
                                          if (n & 1) dp[y] = mma<T, G>(x, vf[c], dp[y]);
                                          else s[y] = mma<T, G>(x, kf[c], s[y]);
                                      });
        const int pu = p0 + i0;                               // position of the unit's first row
        const bool masked = i0 + U > d.Lq || (d.causal && jw + G - 1 > pu);
        float mult = a.sc2, add = 0.f;
        if constexpr (REL) {
            bool near = false;
            if (jw + G - 1 - pu <= -d.reach) add = bias[BIAS_PAD];
            else if (jw - (pu + U - 1) >= d.reach) add = bias[2 * d.reach + BIAS_PAD];
            else near = true;
            if (near) {
                const float* bj = bias + (j - pu - 4 * g + d.reach + BIAS_PAD);
#pragma unroll
                for (int q = 0; q < NB * nq; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[q / nq][4 * (q % nq) + e] = s[q / nq][4 * (q % nq) + e] * mult + bj[-(4 * ng * q + e)];
                mult = 1.f;
            }
        }
#pragma unroll
        for (int q = 0; q < NB * nq; ++q) {
            const int iq = r0 + 4 * ng * q + 4 * g;
            const f32x4 l4 = *reinterpret_cast<const f32x4*>(ls + iq), d4 = *reinterpret_cast<const f32x4*>(ds + iq);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * (q % nq) + e;
                float x = s[q / nq][r] * mult - l4[e];
                if constexpr (REL) x += add;
                s[q / nq][r] = __builtin_amdgcn_exp2f(x);
                dp[q / nq][r] -= d4[e];
            }
        }
        if (masked) {                                         // rows of the unit from `from` on, before the last
            const int from = d.causal ? j - pu : 0, end = d.Lq - i0;
#pragma unroll
            for (int q = 0; q < NB * nq; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = 4 * ng * q + 4 * g + e;
                    const float x = s[q / nq][4 * (q % nq) + e];
                    s[q / nq][4 * (q % nq) + e] = ((k >= from) & (k < end)) ? x : 0.f;
                }
        }
        if (d.drop_p > 0.f) {
#pragma unroll
            for (int q = 0; q < NB * nq; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * (q % nq) + e, k = 4 * ng * q + 4 * g + e;
                    const float keep = drop_keep(a, seed, b, h, i0 + k, j), dl = ds[r0 + k], p = s[q / nq][r];
                    dp[q / nq][r] = p * ((dp[q / nq][r] + dl) * keep - dl);
                    s[q / nq][r] = p * keep;
                }
        } else {
#pragma unroll
            for (int x = 0; x < NB; ++x)
#pragma unroll
                for (int r = 0; r < 4 * nq; ++r) dp[x][r] *= s[x][r];
        }
        if constexpr (REL) {
            // sums over equal distance j - pos: a unit that lies wholly beyond the reach goes to one bucket; otherwise it is written to LDS by
            // diagonals and lane x adds up diagonal x (in a fixed order), whose distance no other lane of the wave holds.
            // Places of a diagonal that the unit does not have stay zero from the start.
            if (jw + G - 1 - pu <= -d.reach || jw - (pu + U - 1) >= d.reach) {
                float z = 0.f;
#pragma unroll
                for (int x = 0; x < NB; ++x)
#pragma unroll
                    for (int r = 0; r < 4 * nq; ++r) z += dp[x][r];
                z = ok ? z : 0.f;
                if (jw < pu) far_back += z; else far_ahead += z;
            } else {
                wave_fence();
                // (row r, key c) at diagonal c - r + U - 1, group of places r / 4, place (c + U - 1) % 4: the 64 writes of a value meet 64 banks
                float* at = skew + (lane % G + U - 1 - 4 * g) * DP + 4 * g + ((lane + U - 1) & 3);
#pragma unroll
                for (int q = 0; q < NB * nq; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) at[4 * ng * q - DP * (4 * ng * q + e)] = ok ? dp[q / nq][4 * (q % nq) + e] : 0.f;
                wave_fence();
                if (lane < DIAG) {
                    const float* row = skew + lane * DP;
                    f32x4 z4 = *reinterpret_cast<const f32x4*>(row);
#pragma unroll
                    for (int r = 4; r < U; r += 4) z4 += *reinterpret_cast<const f32x4*>(row + r);
                    const float z = (z4[0] + z4[1]) + (z4[2] + z4[3]);
                    const int rel = jw - pu + lane - (U - 1);
                    if (rel <= -d.reach) far_back += z;
                    else if (rel >= d.reach) far_ahead += z;
                    else dsum[wave * width + rel + d.reach] += z;
                }
            }
        }
        if constexpr (__is_same(T, _Float16)) {
#pragma unroll
            for (int x = 0; x < NB; ++x)
#pragma unroll
                for (int r = 0; r < 4 * nq; ++r) {
                    dp[x][r] *= rs;
                    s[x][r] *= ps;
                }
        }
        u32x4 pf[PC], df[PC];
#pragma unroll
        for (int c = 0; c < PC; ++c) {
            pf[c] = score_frag<T, G, NB>(s, c);
            df[c] = score_frag<T, G, NB>(dp, c);
        }
        fragment_loop<T, G, PC * MT * 2>([&](int n) __attribute__((always_inline)) { return tf.cols(n & 1 ? qs : gs, (n / 2 % MT) * G, r0, n / 2 / MT); },
                                      [&](int n, u32x4 x) __attribute__((always_inline)) {
                                          const int mt = n / 2 % MT, c = n / 2 / MT;
                                          if (n & 1) dk[mt] = mma<T, G>(x, df[c], dk[mt]);
                                          else dv[mt] = mma<T, G>(x, pf[c], dv[mt]);
                                      });
    };
    // a head's sums: the waves' in order, then the distances of one bucket in ascending order by one thread
    const int rel_lo = j0 - p0 - qtiles * QT, rel_hi = j0 + NW * G - p0;      // distances this workgroup meets
    const int side = d.n_border + 1, nbuckets = side * (d.bidirectional ? 2 : 1);
    auto part_of = [&](int h) { return a.ptab + (((long long)b * d.H + h) * a.tiles * a.splits + tl * a.splits + split) * nbuckets; };
    auto flush = [&](int h) __attribute__((always_inline)) {
        const int lo = max(rel_lo, 1 - d.reach), hi = min(rel_hi, d.reach - 1);
        float* ds = dsum + d.reach;
        far_back = wave_sum(far_back);
        far_ahead = wave_sum(far_ahead);
        if (lane == 0) {
            far[2 * wave] = far_back;
            far[2 * wave + 1] = far_ahead;
        }
        far_back = far_ahead = 0.f;
        __syncthreads();
        for (int x = lo + tid; x <= hi; x += NT)
            for (int wv = 1; wv < NW; ++wv) ds[x] += ds[wv * width + x];
        __syncthreads();
        float* part = part_of(h);
        for (int c = tid; c < nbuckets; c += NT) {
            const bool ahead = d.bidirectional && c >= side;
            const int k = c % side, near = k ? d.border[k - 1] : 0, beyond = k == d.n_border ? d.reach : d.border[k];       // distances near .. beyond - 1
            float x = 0.f;
            if (ahead) for (int r = max(max(near, 1), lo); r <= min(beyond - 1, hi); ++r) x += ds[r];
            else for (int r = max(near, -hi); r <= min(beyond - 1, -lo); ++r) x += ds[-r];
            if (!d.bidirectional && c == 0) for (int r = max(1, lo); r <= hi; ++r) x += ds[r];
            for (int wv = 0; wv < NW; ++wv) {
                if (k == d.n_border) x += far[2 * wv + (ahead ? 1 : 0)];
                if (!d.bidirectional && c == 0) x += far[2 * wv + 1];
            }
            part[c] = x;
        }
        __syncthreads();
    };
    int end = t0;                                             // items before it are copied ahead
    auto tile = [&](int t, const T* qs, const T* gs, const float* ls, const float* ds, T* qn, T* gn, float* ln, float* dn) __attribute__((always_inline)) {
        const int h = kvh * group + t / run, i0 = (first + t % run) * QT;
        settle();
        if (t + 1 < end) fetch(t + 1, qn, gn, ln, dn);
#pragma unroll
        for (int u = 0; u < QT / U; ++u) {
            const int iu = i0 + u * U;
            if (live && iu < d.Lq && !(d.causal && jw > p0 + iu + U - 1)) unit(h, iu, u * U, qs, gs, ls, ds);
        }
    };
    if constexpr (REL) {
        for (int x = lane; x < DIAG * DP; x += 64) skew[x] = 0.f;       // (this wave's own; the first unit is behind a barrier)
    }
    for (int seg = t0; seg < t1; seg = end) {                 // with a bias table head by head: the table and the sums are a head's
        end = REL ? min(t1, (seg / run + 1) * run) : t1;
        if constexpr (REL) {
            fill_bias_range(d, bias, kvh * group + seg / run, rel_lo, rel_hi, tid, NT);
            for (int wv = 0; wv < NW; ++wv)
                for (int x = max(rel_lo, -d.reach) + tid; x <= min(rel_hi, d.reach); x += NT) dsum[wv * width + x + d.reach] = 0.f;
            __syncthreads();
        }
        fetch(seg, q0s, g0s, l0s, d0s);
        for (int t = seg; t < end; t += 2) {
            tile(t, q0s, g0s, l0s, d0s, q1s, g1s, l1s, d1s);
            if (t + 1 < end) tile(t + 1, q1s, g1s, l1s, d1s, q0s, g0s, l0s, d0s);
        }
        if constexpr (REL) flush(kvh * group + seg / run);
    }
    if constexpr (REL) {
        for (int h = kvh * group; h < (kvh + 1) * group; ++h)        // heads this share has not met
            if (t0 >= t1 || h < kvh * group + t0 / run || h > kvh * group + (t1 - 1) / run)
                for (int c = tid; c < nbuckets; c += NT) part_of(h)[c] = 0.f;
    }
    if (j >= d.Lk) return;
    const float f = d.scale / rs, fv = 1.f / ps;
    const long long row = ((long long)b * d.Lk + j) * d.KV * d.dh + (long long)kvh * d.dh;
    const long long n = (long long)d.B * d.Lk * d.KV * d.dh;
#pragma unroll
    for (int q = 0; q < MT * nq; ++q) {
        const int col = 4 * ng * q + 4 * g, r = 4 * (q % nq);
        if (col >= d.dh) continue;
        f32x4 x, y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = ok ? dk[q / nq][r + e] * f : 0.f;
            y[e] = ok ? dv[q / nq][r + e] * fv : 0.f;
        }
        if (a.splits > 1) {
            store4<float>(a.pk + split * n + row + col, x[0], x[1], x[2], x[3]);
            store4<float>(a.pv + split * n + row + col, y[0], y[1], y[2], y[3]);
        } else {
            store4<T>(reinterpret_cast<T*>(d.dk) + row + col, x[0], x[1], x[2], x[3]);
            store4<T>(reinterpret_cast<T*>(d.dv) + row + col, y[0], y[1], y[2], y[3]);
        }
    }
}

// out[n] = sum of `splits` partial outputs, in order (n a multiple of 4)
template <typename T>
__global__ __launch_bounds__(256) void attn_sum_kernel(const float* part, T* out, long long n, int splits) {
    for (long long x = 4 * ((long long)blockIdx.x * 256 + threadIdx.x); x < n; x += 4ll * 256 * gridDim.x) {
        f32x4 s = *reinterpret_cast<const f32x4*>(part + x);
        for (int k = 1; k < splits; ++k) s += *reinterpret_cast<const f32x4*>(part + k * n + x);
        store4<T>(out + x, s[0], s[1], s[2], s[3]);
    }
}
// delta += the shares of its correction, in order
__global__ __launch_bounds__(256) void attn_delta_kernel(const float* eps, float* delta, long long n, int splits) {
    for (long long x = (long long)blockIdx.x * 256 + threadIdx.x; x < n; x += 256ll * gridDim.x) {
        float s = delta[x];
        for (int k = 0; k < splits; ++k) s += eps[k * n + x];
        delta[x] = s;
    }
}
// dtable[c][h] = sum over samples and key blocks, one wave per entry, fixed order
__global__ __launch_bounds__(64) void attn_table_kernel(const AttnArgs a, int nb) {
    const int c = blockIdx.x % nb, h = blockIdx.x / nb, lane = threadIdx.x, parts = a.tiles * a.splits;
    float s = 0.f;
    const int n = a.d.B * parts;
    for (int x = lane; x < n; x += 64) s += a.ptab[(((long long)(x / parts) * a.d.H + h) * parts + x % parts) * nb + c];
    s = wave_sum(s);
    if (lane) return;
    const long long o = (long long)c * a.d.H + h;
    if (a.d.table_dtype == EKAID_F32) reinterpret_cast<float*>(a.d.dtable)[o] = s;
    else if (a.d.table_dtype == EKAID_BF16) reinterpret_cast<__bf16*>(a.d.dtable)[o] = (__bf16)s;
    else reinterpret_cast<_Float16*>(a.d.dtable)[o] = (_Float16)s;
}

struct BwdPlan {
    int gq, nwq, tq, sq;        // dq: block edge, waves, row tiles, splits
    int gk, nwk, tk, sk;        // dk / dv
    size_t delta, nrm, vn, eps, tab, po, pk, total;      // float offsets
    int v_parts;
};
static size_t align4(size_t n) { return (n + 3) & ~(size_t)3; }

static BwdPlan bwd_plan(const ekaid_attn_t* a) {
    BwdPlan p;
    const int esz = a->dtype == EKAID_F32 ? 4 : 2;
    // blocks of 32 x 32 halve the LDS reads a product; blocks of 16 x 16 where those of 32 leave registers for one wave a SIMD only (dk, dv of
    // 128-wide 16-bit heads, before the table's sums joined them: 320 -> 275 us for 16 heads x 2048 causal; 64 wide it is 161 against 204 us)
    // and for few rows
    p.gq = a->Lq <= 64 || (esz == 4 && a->dh > 128) ? 16 : 32;
    p.nwq = p.gq == 32 ? 4 : waves_for_rows(a->Lq, esz == 4 && a->dh > 128);
    p.tq = cdiv(a->Lq, p.gq * p.nwq);
    p.gk = a->Lk <= 64 || a->dh > (esz == 4 ? 128 : 64) ? 16 : 32;
    p.nwk = p.gk == 32 ? 4 : waves_for_rows(a->Lk, esz == 4 && a->dh > 128);
    p.tk = cdiv(a->Lk, p.gk * p.nwk);
    auto split = [](long long wgs, int waves, int work) {
        const long long want = 4 * 512 / waves;
        long long s = wgs > 0 && wgs < want / 2 ? (want + wgs - 1) / wgs : 1;
        if (s > (work + 1) / 2) s = (work + 1) / 2;
        return (int)(s < 1 ? 1 : s);
    };
    p.sq = split((long long)a->B * a->H * p.tq, p.nwq, cdiv(a->Lk, attn_kt(esz, a->dh, p.gq)));
    p.sk = split((long long)a->B * a->KV * p.tk, p.nwk, cdiv(a->Lq, attn_kt(esz, a->dh, p.gk)) * (a->H / a->KV));
    const size_t rows = (size_t)a->B * a->H * a->Lq, bh = (size_t)a->B * a->H;
    const int nb = a->table ? (a->n_border + 1) * (a->bidirectional ? 2 : 1) : 0;
    size_t o = 0;
    p.delta = o; o += align4(rows);
    p.nrm = o; o += align4(bh * p.tq * p.sq);
    // (value norms: some 2048 workgroups, 64 rows or more each)
    p.v_parts = a->dtype == EKAID_F16 ? std::min(cdiv(a->Lk, 64), std::max(1, std::min(64, 2048 / std::max(1, a->B * a->KV)))) : 0;
    p.vn = o; o += align4((size_t)a->B * a->KV * p.v_parts);
    p.eps = o; o += a->table && p.sq > 1 ? align4(rows * p.sq) : 0;
    p.tab = o; o += align4(bh * p.tk * p.sk * nb);
    p.po = o; o += p.sq > 1 ? p.sq * rows * a->dh : 0;
    p.pk = o; o += p.sk > 1 ? 2 * p.sk * (size_t)a->B * a->Lk * a->KV * a->dh : 0;
    p.total = o * sizeof(float);
    return p;
}
size_t attn_bwd_workspace(const ekaid_attn_t* a) { return bwd_plan(a).total; }

template <typename T, int DH, int G, int NW, bool REL> static int launch_dq(const AttnArgs& a, hipStream_t st) {
    constexpr int KT = attn_kt((int)sizeof(T), DH, G);
    const size_t lds = 4 * NW + 4 * KT + (REL ? 4 * (2 * (a.d.reach + BIAS_PAD) + 1) : 0);
    if (int rc = attn_lds_limit((const void*)attn_dq_kernel<T, DH, G, NW, KT, REL>, 96 * 1024)) return rc;
    hipLaunchKernelGGL((attn_dq_kernel<T, DH, G, NW, KT, REL>), dim3(a.d.B * a.d.H * a.tiles * a.splits), dim3(64 * NW), lds, st, a);
    return check_launch("attn_dq");
}
template <typename T, int DH, bool REL> static int pick_dq(const AttnArgs& a, const BwdPlan& p, hipStream_t st) {
    if constexpr (!(sizeof(T) == 4 && DH > 128))
        if (p.gq == 32) return launch_dq<T, DH, 32, 4, REL>(a, st);
    if (p.nwq == 1) return launch_dq<T, DH, 16, 1, REL>(a, st);
    if (p.nwq == 2) return launch_dq<T, DH, 16, 2, REL>(a, st);
    return launch_dq<T, DH, 16, 4, REL>(a, st);
}
template <typename T, int DH, int G, int NW, bool REL> static int launch_dkv(const AttnArgs& a, hipStream_t st) {
    constexpr int QT = attn_kt((int)sizeof(T), DH, G);
    constexpr int U = QT < 32 ? QT : 32;
    const size_t lds = REL ? 4 * ((size_t)(NW + 1) * (2 * a.d.reach + 1) + 2 * BIAS_PAD + 2 * NW + 4 + NW * (U + G - 1) * (U + 4)) : 0;
    if (int rc = attn_lds_limit((const void*)attn_dkv_kernel<T, DH, G, NW, QT, REL>, 92 * 1024)) return rc;
    hipLaunchKernelGGL((attn_dkv_kernel<T, DH, G, NW, QT, REL>), dim3(a.d.B * a.d.KV * a.tiles * a.splits), dim3(64 * NW), lds, st, a);
    return check_launch("attn_dkv");
}
template <typename T, int DH, bool REL> static int pick_dkv(const AttnArgs& a, const BwdPlan& p, hipStream_t st) {
    if constexpr (DH <= (sizeof(T) == 4 ? 128 : 64))
        if (p.gk == 32) return launch_dkv<T, DH, 32, 4, REL>(a, st);
    if (p.nwk == 1) return launch_dkv<T, DH, 16, 1, REL>(a, st);
    if (p.nwk == 2) return launch_dkv<T, DH, 16, 2, REL>(a, st);
    return launch_dkv<T, DH, 16, 4, REL>(a, st);
}
template <typename T> static int sum_parts(const float* part, void* out, long long n, int splits, hipStream_t st) {
    hipLaunchKernelGGL(attn_sum_kernel<T>, dim3((int)std::min<long long>((n / 4 + 255) / 256, 4096)), dim3(256), 0, st, part, (T*)out, n, splits);
    return check_launch("attn_sum");
}
template <typename T> static int run_bwd(AttnArgs a, const BwdPlan& p, hipStream_t st) {
    const ekaid_attn_t& d = a.d;
    int rc = EKAID_OK;
    a.gp = a.near = 1;
    a.tiles = p.tq;
    a.splits = p.sq;
    a.dq_parts = p.tq * p.sq;
    if (p.v_parts) {
        hipLaunchKernelGGL(attn_vnorm_kernel, dim3(d.B * d.KV * p.v_parts), dim3(256), 0, st, a);
        if ((rc = check_launch("attn_vnorm"))) return rc;
    }
    if (d.table)
        rc = d.dh <= 64 ? pick_dq<T, 64, true>(a, p, st) : d.dh <= 128 ? pick_dq<T, 128, true>(a, p, st) : pick_dq<T, 256, true>(a, p, st);
    else
        rc = d.dh <= 64 ? pick_dq<T, 64, false>(a, p, st) : d.dh <= 128 ? pick_dq<T, 128, false>(a, p, st) : pick_dq<T, 256, false>(a, p, st);
    if (rc) return rc;
    if (p.sq > 1 && (rc = sum_parts<T>(a.po, d.dq, (long long)d.B * d.Lq * d.H * d.dh, p.sq, st))) return rc;
    if (d.table && p.sq > 1) {
        const long long n = (long long)d.B * d.H * d.Lq;
        hipLaunchKernelGGL(attn_delta_kernel, dim3((int)std::min<long long>((n + 255) / 256, 4096)), dim3(256), 0, st, a.eps, a.delta, n, p.sq);
        if ((rc = check_launch("attn_delta"))) return rc;
    }
    const int nb = (d.n_border + 1) * (d.bidirectional ? 2 : 1);
    a.tiles = p.tk;                                           // (no keys: no key tiles, the table's sums are of nothing)
    a.splits = p.sk;
    if (d.table && d.Lk == 0) {
        hipLaunchKernelGGL(attn_table_kernel, dim3(nb * d.H), dim3(64), 0, st, a, nb);
        return check_launch("attn_table");
    }
    if (d.Lk == 0) return EKAID_OK;
    if (d.table)
        rc = d.dh <= 64 ? pick_dkv<T, 64, true>(a, p, st) : d.dh <= 128 ? pick_dkv<T, 128, true>(a, p, st) : pick_dkv<T, 256, true>(a, p, st);
    else
        rc = d.dh <= 64 ? pick_dkv<T, 64, false>(a, p, st) : d.dh <= 128 ? pick_dkv<T, 128, false>(a, p, st) : pick_dkv<T, 256, false>(a, p, st);
    if (rc) return rc;
    if (d.table) {
        hipLaunchKernelGGL(attn_table_kernel, dim3(nb * d.H), dim3(64), 0, st, a, nb);
        if ((rc = check_launch("attn_table"))) return rc;
    }
    if (p.sk == 1) return EKAID_OK;
    const long long n = (long long)d.B * d.Lk * d.KV * d.dh;
    if ((rc = sum_parts<T>(a.pk, d.dk, n, p.sk, st))) return rc;
    return sum_parts<T>(a.pv, d.dv, n, p.sk, st);
}
}  // namespace ekaid

extern "C" int ekaid_attn_bwd(const ekaid_attn_t* a, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace ekaid;
    if (int rc = attn_check(a, "attn_bwd")) return rc;
    if (a->B == 0 || a->Lq == 0) { set_error("attn_bwd: no query rows (the caller zeroes dk, dv, dtable)"); return EKAID_ERR_ARG; }
    if (!a->q || !a->out || !a->dout || !a->lse || !a->dq || (a->table && !a->dtable) || (a->Lk && (!a->k || !a->v || !a->dk || !a->dv))) {
        set_error("attn_bwd: null operand");
        return EKAID_ERR_ARG;
    }
    if (((uintptr_t)a->dout | (uintptr_t)a->out | (uintptr_t)a->out32) & 15) { set_error("attn_bwd: operands must be 16-byte aligned"); return EKAID_ERR_ARG; }
    const BwdPlan p = bwd_plan(a);
    if (!workspace || workspace_bytes < p.total) { set_error("attn_bwd: workspace of %zu bytes needed", p.total); return EKAID_ERR_ARG; }
    AttnArgs k = {};
    k.d = *a;
    k.seed = DS(a->drop_seed);
    k.inv_keep = 1.f / (1.f - a->drop_p);
    k.sc2 = a->scale * LOG2E;
    float* w = (float*)workspace;
    k.delta = w + p.delta;
    k.nrm = w + p.nrm;
    k.vn = w + p.vn;
    k.v_parts = p.v_parts;
    (void)frexpf(k.inv_keep, &k.keep_exp);
    if (k.inv_keep == ldexpf(1.f, k.keep_exp - 1)) --k.keep_exp;
    k.eps = w + p.eps;
    k.ptab = w + p.tab;
    k.po = w + p.po;
    k.pk = w + p.pk;
    k.pv = k.pk + (size_t)p.sk * a->B * a->Lk * a->KV * a->dh;
    hipStream_t st = (hipStream_t)stream;
    return a->dtype == EKAID_F32 ? run_bwd<float>(k, p, st) : a->dtype == EKAID_BF16 ? run_bwd<__bf16>(k, p, st) : run_bwd<_Float16>(k, p, st);
}
