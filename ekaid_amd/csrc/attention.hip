// Forward of the attention operators (include/ekaid_hip.h: ekaid_attn_t): one pass over the keys with the running maximum and sum.
#include "attn.h"

namespace ekaid {

// running maximum / sum: returns the factor that earlier sums and outputs take
template <int G, int NB>
__device__ __forceinline__ float online_softmax(typename Blk<G>::acc (&s)[NB], float& m, float& l) {
    constexpr int nv = 4 * Blk<G>::nq;
    float mx = m;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < nv; ++r) mx = fmaxf(mx, s[b][r]);
    mx = across_groups_max<G>(mx);
    const float base = mx == NEG_INF ? 0.f : mx;          // nothing valid yet: every power below is 2^-inf = 0
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    float t = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < nv; ++r) {
            s[b][r] = __builtin_amdgcn_exp2f(s[b][r] - base);
            t += s[b][r];
        }
    l = l * alpha + t;                                    // this lane's keys only; the lane groups meet at the end
    m = mx;
    return alpha;
}

template <int G, int NB>
__device__ __forceinline__ void drop_scores(const AttnArgs& a, typename Blk<G>::acc (&s)[NB], int b, int h, int i, int j0, int lane) {
    constexpr int ng = Blk<G>::ng, nq = Blk<G>::nq;
    const uint64_t seed = drop_seed_value(a.seed);
#pragma unroll
    for (int q = 0; q < NB * nq; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[q / nq][4 * (q % nq) + e] *= drop_keep(a, seed, b, h, i, j0 + 4 * ng * q + 4 * (lane / G) + e);
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
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* p = reinterpret_cast<T*>(a.d.out) + ((long long)w.b * a.d.Lq + i) * a.d.H * a.d.dh + (long long)h * a.d.dh;
#pragma unroll
    for (int q = 0; q < DH / G * nq; ++q) {
        const int col = 4 * ng * q + 4 * g;
        const auto& t = o[q / nq];
        if (col < a.d.dh) store4<T>(p + col, t[4 * (q % nq)] * inv, t[4 * (q % nq) + 1] * inv, t[4 * (q % nq) + 2] * inv, t[4 * (q % nq) + 3] * inv);
    }
    if (g == 0 && a.d.lse) a.d.lse[row] = l == 0.f ? POS_INF : m + __builtin_amdgcn_logf(l);
}

// ---- few query rows (a new token; the heads that share keys packed into the rows): key tiles through registers into LDS
template <typename T, int DH, int G, int NW, int KT>
__global__ __launch_bounds__(64 * NW) void attn_fwd_kernel(const AttnArgs a) {
    constexpr int NT = 64 * NW, NB = KT / G, NC = DH / (Elem<T>::epl * Blk<G>::ng), PC = KT / (Elem<T>::epl * Blk<G>::ng), MT = DH / G;
    constexpr int LDK = Ld<T, DH>::row, LDV = Ld<T, DH>::col;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* Ks = reinterpret_cast<T*>(smem);
    T* Vs = Ks + KT * LDK;
    unsigned char* kms = reinterpret_cast<unsigned char*>(Vs + KT * LDV);
    float* bias = reinterpret_cast<float*>(kms + KT);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const RowWork w(a);
    const ekaid_attn_t& d = a.d;
    const int R = d.Lq * a.gp, r = (w.tile * NW + wave) * G + lane % G;
    const bool ok = r < R;
    const int i = ok ? r / a.gp : 0, hg = ok ? r % a.gp : 0, h = w.head0 + hg;
    const int p0 = query_pos(d, w.b), pos = p0 + i;
    const int len = key_len(d, w.b);
    int kend = len;
    if (d.causal) {
        const int last = min(R, (w.tile + 1) * NW * G) - 1;
        kend = max(0, min(len, p0 + last / a.gp + 1));
    }
    const int nt = (kend + KT - 1) / KT, per = (nt + a.splits - 1) / a.splits, t0 = w.split * per, t1 = min(nt, t0 + per);
    const unsigned char* mask = d.key_mask ? d.key_mask + w.b * d.mask_batch : nullptr;
    if (d.table) fill_bias(d, bias, w.head0, a.gp, 0, tid, NT);

    u32x4 qf[NC];
    const T* qrow = reinterpret_cast<const T*>(d.q) + w.b * d.q_batch + i * d.q_row + (long long)h * d.dh;
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = row_frag_global<T, G>(qrow, c, d.dh, ok, lane);

    const T* kb = reinterpret_cast<const T*>(d.k) + w.b * d.k_batch + (long long)w.kvh * d.dh;
    const T* vb = reinterpret_cast<const T*>(d.v) + w.b * d.v_batch + (long long)w.kvh * d.dh;
    Stage<T, DH, KT, NT> sk, sv;
    typename Blk<G>::acc o[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[mt] = zero_acc<G>();
    float m = NEG_INF, l = 0.f;
    if (t0 < t1) {
        sk.load(kb, d.k_row, t0 * KT, len, d.dh, mask, tid);
        sv.load(vb, d.v_row, t0 * KT, len, d.dh, mask, tid);
    }
    for (int t = t0; t < t1; ++t) {
        sk.store(Ks, LDK, tid);
        sv.store(Vs, LDV, tid);
        if (mask) for (int j = tid; j < KT; j += NT) kms[j] = t * KT + j < len ? mask[t * KT + j] : 0;
        __syncthreads();
        if (t + 1 < t1) {
            sk.load(kb, d.k_row, (t + 1) * KT, len, d.dh, mask, tid);
            sv.load(vb, d.v_row, (t + 1) * KT, len, d.dh, mask, tid);
        }
        typename Blk<G>::acc s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            s[b] = zero_acc<G>();
#pragma unroll
            for (int c = 0; c < NC; ++c) s[b] = mma<T, G>(row_frag<T, G>(Ks, LDK, b * G, c, lane), qf[c], s[b]);
        }
        const bool partial = mask || (t + 1) * KT > len || (d.causal && (t + 1) * KT > p0 + (w.tile * NW * G) / a.gp + 1);
        finish_scores<G, NB>(a, s, t * KT, len, pos, d.table ? bias + hg * (2 * d.reach + 1) : nullptr, mask ? kms : nullptr, partial, lane);
        const float alpha = online_softmax<G, NB>(s, m, l);
        if (d.drop_p > 0.f) drop_scores<G, NB>(a, s, w.b, h, i, t * KT, lane);
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4 * Blk<G>::nq; ++e) o[mt][e] *= alpha;
        }
#pragma unroll
        for (int c = 0; c < PC; ++c) {
            const u32x4 pf = score_frag<T, G, NB>(s, c);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) o[mt] = mma<T, G>(col_frag<T, G>(Vs, LDV, mt * G, c, lane), pf, o[mt]);
        }
        __syncthreads();
    }
    write_rows<T, DH, G>(a, w, o, m, l, i, h, ok, lane);
}

// ---- many query rows: NW * G rows a workgroup, key tiles copied to LDS one tile ahead of the products
template <typename T, int DH, int G, int NW, int KT>
__global__ __launch_bounds__(64 * NW, DH * (int)sizeof(T) * G > 8192 ? 1 : 2) void attn_tile_fwd_kernel(const AttnArgs a) {
    constexpr int NT = 64 * NW, NB = KT / G, NC = DH / (Elem<T>::epl * Blk<G>::ng), PC = KT / (Elem<T>::epl * Blk<G>::ng), MT = DH / G, nv = 4 * Blk<G>::nq;
    __shared__ __attribute__((aligned(16))) T k0[KT * DH], k1[KT * DH], v0[KT * DH], v1[KT * DH];
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* bias = reinterpret_cast<float*>(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const RowWork w(a);
    const ekaid_attn_t& d = a.d;
    const int row0 = (w.tile * NW + wave) * G, h = w.head0;
    const bool ok = row0 + lane % G < d.Lq, live = row0 < d.Lq;
    const int i = min(row0 + lane % G, d.Lq - 1), p0 = query_pos(d, w.b), pos = p0 + i, pmin = p0 + min(row0, d.Lq - 1), pmax = p0 + min(row0 + G, d.Lq) - 1;
    const int len = key_len(d, w.b), kend = d.causal ? max(0, min(len, p0 + min(d.Lq, (w.tile + 1) * NW * G))) : len;
    const int nt = (kend + KT - 1) / KT, per = (nt + a.splits - 1) / a.splits, t0 = w.split * per, t1 = min(nt, t0 + per);
    const int width = d.table ? 2 * (d.reach + BIAS_PAD) + 1 : 0;
    if (d.table) {
        fill_bias(d, bias, h, 1, BIAS_PAD, tid, NT);
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
        ck.issue(k0, t0 * KT, len, d.dh, ring.tile(t0), wave);
        cv.issue(v0, t0 * KT, len, d.dh, ring.tile(t0), wave);
    }
    auto tile = [&](int t, const T* ks, const T* vs, T* kn, T* vn) __attribute__((always_inline)) {
        settle();
        ring.step(t);
        if (t + 1 < t1) {
            ck.issue(kn, (t + 1) * KT, len, d.dh, ring.tile(t + 1), wave);
            cv.issue(vn, (t + 1) * KT, len, d.dh, ring.tile(t + 1), wave);
        }
        if (!live || (d.causal && t * KT > pmax)) return;
        if constexpr (DH * sizeof(T) > 128) tf.refresh();
        typename Blk<G>::acc s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b] = zero_acc<G>();
        fragment_loop<T, NC * NB>([&](int n) __attribute__((always_inline)) { return tf.rows(ks, (n % NB) * G, n / NB); },
                                  [&](int n, u32x4 x) __attribute__((always_inline)) { s[n % NB] = mma<T, G>(x, qf[n / NB], s[n % NB]); });
        const Affine f = scores_by_row<G, NB>(a, s, t * KT, len, pos, pmin, pmax, d.table ? bias : nullptr, ring.tile(t), lane);
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < nv; ++r) mx = fmaxf(mx, s[b][r]);
        const float mn = fmaxf(m, across_groups_max<G>(mx) * f.mult + f.add);      // (mult >= 0)
        const float base = mn == NEG_INF ? 0.f : mn, shift = f.add - base;
        if (__any(mn != m)) {
            const float alpha = __builtin_amdgcn_exp2f(m - base);
            l *= alpha;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < nv; ++e) o[mt][e] *= alpha;
        }
        m = mn;
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
        fragment_loop<T, PC * MT>([&](int n) __attribute__((always_inline)) { return tf.cols(vs, (n % MT) * G, 0, n / MT); },
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
    const float inv = l == 0.f ? 0.f : 1.f / l;
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
        store4<T>(out + c, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
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
    if ((long long)a->B * a->H * ((long long)a->Lq + a->Lk + 64) > (1ll << 33) || (long long)a->B * a->H > (1 << 24)) {
        set_error("%s: too many rows for one launch", who);
        return EKAID_ERR_UNSUPPORTED;
    }
    return EKAID_OK;
}

struct FwdPlan { int few, g, nw, gp, tiles, splits, kt; size_t ws; };

// Waves of 16 rows: as few rows as possible beyond R (a wave on rows that do not exist costs as much as one on rows that do)
int waves_for_rows(int R) {
    int best = 4, cost = 1 << 30;
    for (int nw = 4; nw >= 1; nw >>= 1) {
        const int c = cdiv(R, 16 * nw) * 16 * nw * (nw == 4 ? 8 : nw == 2 ? 9 : 12);      // smaller workgroups copy the tiles more often
        if (c < cost) { cost = c; best = nw; }
    }
    return best;
}

static FwdPlan fwd_plan(const ekaid_attn_t* a) {
    FwdPlan p;
    const int group = a->H / a->KV;
    const bool wide32 = a->dtype == EKAID_F32 && a->dh > 128;
    p.few = a->Lq < 17;
    p.gp = p.few && group > 1 && (!a->table || group * (2 * a->reach + 1) <= 8192) ? group : 1;
    const int R = a->Lq * p.gp;
    if (p.few) {
        p.g = R <= 64 || wide32 ? 16 : 32;
        p.nw = R <= 16 ? 1 : R <= 32 && p.g == 16 ? 2 : 4;
        if (wide32 && p.nw == 1) p.nw = 2;      // one wave would have to hold a whole staged tile: it spills
        p.kt = a->dh > 128 || (a->dtype == EKAID_F32 && a->dh > 64) ? 32 : 64;
    } else {
        p.g = R <= 64 || wide32 ? 16 : 32;
        p.nw = p.g == 32 ? 4 : waves_for_rows(R);
        p.kt = attn_kt(a->dtype == EKAID_F32 ? 4 : 2, a->dh, p.g);
    }
    p.tiles = cdiv(R, p.g * p.nw);
    const long long wgs = (long long)a->B * (a->H / p.gp) * p.tiles;
    const int key_tiles = cdiv(a->Lk, p.kt);
    long long s = 1;
    const long long want = 4 * 512 / p.nw;
    if (wgs < want / 2 && key_tiles > 1) s = (want + wgs - 1) / (wgs > 0 ? wgs : 1);
    if (s > (key_tiles + 1) / 2) s = (key_tiles + 1) / 2;
    if (s < 1) s = 1;
    p.splits = (int)s;
    p.ws = p.splits > 1 ? (size_t)p.splits * a->B * a->H * a->Lq * (a->dh + 2) * sizeof(float) : 0;
    return p;
}

template <typename T, int DH, int G, int NW, int KT> static int launch_few(const AttnArgs& a, int grid, hipStream_t st) {
    constexpr size_t base = (size_t)KT * (Ld<T, DH>::row + Ld<T, DH>::col) * sizeof(T) + KT;
    const size_t lds = base + (a.d.table ? (size_t)a.gp * (2 * a.d.reach + 1) * 4 : 0);
    if (int rc = attn_lds_limit((const void*)attn_fwd_kernel<T, DH, G, NW, KT>, 160 * 1024)) return rc;
    hipLaunchKernelGGL((attn_fwd_kernel<T, DH, G, NW, KT>), dim3(grid), dim3(64 * NW), lds, st, a);
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
    if (p.few) {
        constexpr int KT = DH > 128 || (sizeof(T) == 4 && DH > 64) ? 32 : 64;
        if constexpr (!(sizeof(T) == 4 && DH > 128)) {
            if (p.g == 32) return launch_few<T, DH, 32, 4, KT>(a, grid, st);
            if (p.nw == 1) return launch_few<T, DH, 16, 1, KT>(a, grid, st);
        }
        if (p.nw == 2) return launch_few<T, DH, 16, 2, KT>(a, grid, st);
        return launch_few<T, DH, 16, 4, KT>(a, grid, st);
    }
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
    k.tiles = p.tiles;
    k.splits = p.splits;
    k.po = (float*)workspace;
    k.pml = k.po + (size_t)p.splits * a->B * a->H * a->Lq * a->dh;
    hipStream_t st = (hipStream_t)stream;
    return a->dtype == EKAID_F32 ? run_fwd<float>(k, p, st) : a->dtype == EKAID_BF16 ? run_fwd<__bf16>(k, p, st) : run_fwd<_Float16>(k, p, st);
}
