// Linear attention with one decay per head: a recurrence over time whose state is a Dk x Dv matrix per head,
//     S_t = e^g S_{t-1} + k_t v_t^T,    o_t = scale * q_t S_t,    g <= 0 per head.
// The backward pass is the same recurrence on other operands (do = the gradient of o, P = the gradient of the last state):
//     dq = the forward recurrence on (do, v, k);  dk = the recurrence from the end on (v, do, q);  dv = the one from the end on (k, q, do),
// where a step from the end adds, reads and then decays (R = P + scale q do^T, out, P = e^g R): the gradient of the last state reaches the last
// token undecayed, and what is left in front of the first token is the gradient of the first state.
#include "common.h"

namespace {

struct LinAttnArgs {
    const void *q, *k, *v;
    void* o;
    const float* g;              // [H] log decay
    const float* s_in;           // [B][H] states, strides s_h (one head), element (i, j) at i * s_i + j * s_j; nullptr = zero
    float* s_out;                // the same layout as s_in, or nullptr
    const int* lengths;          // [B] tokens of each sequence, or nullptr = T
    long qb, qt, qh, kb, kt, kh, vb, vt, vh, ob, ot, oh;      // element strides of batch row, token and head (inner stride 1)
    int B, T, H, Dk, Dv, rq, rk, rv;                          // head h reads head h / rq of q, h / rk of k, h / rv of v
    int si, sj;
    float oscale, uscale;        // on what is read, on what is added
    int rev;
};

template <typename T> __device__ __forceinline__ void st1(T* p, long i, float v);
template <> __device__ __forceinline__ void st1<float>(float* p, long i, float v) { p[i] = v; }
template <> __device__ __forceinline__ void st1<b16>(b16* p, long i, float v) {
    unsigned h, l;
    split2_bf16(v, 0.f, h, l);
    p[i] = (b16)(h & 0xffff);
}

// ---- chunked form --------------------------------------------------------------------------------------------------------------------------
// C tokens at a time (fp32: 32, bf16: 64), positions i, j inside the chunk, e = 1 forward and 0 from the end:
//     o_i = e^{g (i + e)} q_i S + sum_{j <= i} e^{g (i - j)} (q_i k_j) v_j,        S <- e^{g C} S + sum_j e^{g (C - e - j)} k_j v_j^T
// A workgroup owns a (batch row, head, segment of the time axis); its waves split the columns of v, each keeps its Dk x DVW slice of S in MFMA
// accumulators for the whole segment.  The accumulator layout (column = lane & 15, row = 4 (lane >> 4) + i) is that of an operand whose k runs along
// the rows, up to an order of k that both operands may share: S and the scores k q^T go from accumulators into the next product without
// touching LDS.  Every wave forms the scores for itself (a fifth of its products) rather than meet the others at a barrier.
//     o^T = S^T q^T + v^T (k q^T):  a lane ends with 4 consecutive columns of one token.
// fp32 operands run on the fp32 MFMA.  bf16 operands are exact as they are; what is computed is split into bf16 pieces: S and the scores, which
// only reach the bf16 result, into two (2^-17), the decayed v that is added to S into three (all 24 bits: S stays fp32-exact).
// The decay of S is S + S (e^{gC} - 1): a factor rounded to fp32 is off the same way in every chunk, 1e-4 of a state with a memory of 2^12 tokens.
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t* lds4_t;

template <typename T> struct Mma;
template <> struct Mma<float> {
    typedef f32x4 Frag;
    static constexpr int C = 32, KB = 16, PADK = 16, NS = 1, NV = 1;      // chunk, k per fragment, LDS row padding, pieces of S / scores and of v
    // row m of a score tile is token 4 (m & 3) + (m >> 2): the column reads below then take four neighbouring rows at once, without bank conflicts
    __device__ __forceinline__ static int srow(int g, int i) { return 4 * i + g; }
    __device__ __forceinline__ static int krow(int m) { return 4 * (m & 3) + (m >> 2); }
    __device__ __forceinline__ static f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    __device__ __forceinline__ static Frag row(const float* p, int ld, int r, int u, int g) { return *reinterpret_cast<const f32x4*>(p + r * ld + 16 * u + 4 * g); }
    __device__ __forceinline__ static Frag col(const float* p, int ld, int c0, int u, int lane) {
        Frag f;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = p[(16 * u + 4 * i + (lane >> 4)) * ld + c0 + (lane & 15)];
        return f;
    }
    template <int N> __device__ __forceinline__ static void pieces(const f32x4* x, Frag* out) { out[0] = x[0]; }
    __device__ __forceinline__ static void scaled(Frag f, const float* w, f32x4* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[0][i] = f[i] * w[i];
    }
};
template <> struct Mma<b16> {
    typedef bf16x8_t Frag;
    static constexpr int C = 64, KB = 32, PADK = 16, NS = 2, NV = 3;
    __device__ __forceinline__ static int srow(int g, int i) { return 4 * g + i; }
    __device__ __forceinline__ static int krow(int m) { return m; }
    __device__ __forceinline__ static f32x4 mma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    __device__ __forceinline__ static Frag row(const b16* p, int ld, int r, int u, int g) {
        const s16x4_t a = *reinterpret_cast<const s16x4_t*>(p + r * ld + 32 * u + 4 * g), b = *reinterpret_cast<const s16x4_t*>(p + r * ld + 32 * u + 16 + 4 * g);
        return __builtin_bit_cast(bf16x8_t, (s16x8_t)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    // transpose reads: 16 lanes read a [4 rows][16 columns] block row-major, each gets the 4 rows of its own column
    __device__ __forceinline__ static Frag col(const b16* p, int ld, int c0, int u, int lane) {
        const b16* q = p + (32 * u + 4 * (lane >> 4) + ((lane & 15) >> 2)) * ld + c0 + 4 * (lane & 3);
        const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(__attribute__((address_space(3))) const b16*)q);
        const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(__attribute__((address_space(3))) const b16*)(q + 16 * ld));
        return __builtin_bit_cast(bf16x8_t, (s16x8_t)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    template <int N> __device__ __forceinline__ static void pieces(const f32x4* x, Frag* out) {
        u32x4_t w[N];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            unsigned p[3];
            splitn_bf16<N>(x[j >> 1][2 * (j & 1)], x[j >> 1][2 * (j & 1) + 1], p);
#pragma unroll
            for (int n = 0; n < N; ++n) w[n][j] = p[n];
        }
#pragma unroll
        for (int n = 0; n < N; ++n) out[n] = __builtin_bit_cast(bf16x8_t, w[n]);
    }
    __device__ __forceinline__ static void scaled(Frag f, const float* w, f32x4* x) {
        const u32x4_t u = __builtin_bit_cast(u32x4_t, f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j >> 1][2 * (j & 1)] = __uint_as_float(u[j] << 16) * w[2 * j];
            x[j >> 1][2 * (j & 1) + 1] = __uint_as_float(u[j] & 0xffff0000u) * w[2 * j + 1];
        }
    }
};

// 16 bytes of a row: `left` elements of it exist; `vec`: rows are whole 16-byte pieces
template <typename T> __device__ __forceinline__ u32x4_t load16(const T* p, bool vec, int left) {
    constexpr int E = 16 / sizeof(T);
    u32x4_t r = {0u, 0u, 0u, 0u};
    if (left <= 0) return r;
    if (vec) return *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (j < left) {
            if constexpr (sizeof(T) == 4) r[j] = __float_as_uint(p[j]);
            else r[j >> 1] |= (unsigned)p[j] << (16 * (j & 1));
        }
    return r;
}

template <typename T, int D, int NT> struct Stage {            // a chunk of one operand: registers on the way from memory to LDS
    static constexpr int E = 16 / sizeof(T), V = D / E, N = Mma<T>::C * V / NT, LD = D + Mma<T>::PADK;
    static_assert(N * NT == Mma<T>::C * V, "a chunk is a whole number of pieces per thread");
    u32x4_t r[N];
    // rows: token `first` and on in steps of `step` elements (negative from the end); n of them exist
    __device__ __forceinline__ void load(const T* first, long step, int n, int dim, bool vec) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int x = threadIdx.x + j * NT, row = x / V, c = x % V * E;
            r[j] = load16(first + row * step + c, vec, row < n ? dim - c : 0);
        }
    }
    __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int x = threadIdx.x + j * NT;
            *reinterpret_cast<u32x4_t*>(lds + x / V * LD + x % V * E) = r[j];
        }
    }
};

struct ChunkArgs {
    LinAttnArgs a;
    float* seg_state;            // [B * H][nseg - 1][Dk * Dv]: a segment's own contribution, after the scan the state that enters the next one
    int nseg, seg_len;           // segments of seg_len tokens (a multiple of the chunk)
    int vq, vk, vv, vo;          // 16-byte accesses possible
};

__device__ __forceinline__ float decay_power(float g, int n) { return n == 0 ? 1.f : expf(g * (float)n); }

// STATE_ONLY: the segment's own contribution to the state (from zero), nothing is read of q and no o is written
template <typename T, typename TO, int DKP, int DVP, bool STATE_ONLY>
__global__ __launch_bounds__((DVP < 64 ? DVP / 16 : 4) * 64) void linattn_chunk_kernel(const ChunkArgs ca) {
    typedef Mma<T> M;
    constexpr int NW = DVP < 64 ? DVP / 16 : 4, NT = NW * 64, DVW = DVP / NW, C = M::C, KB = M::KB, TPF = KB / 16;
    constexpr int KT = DKP / 16, KF = DKP / KB, VT = DVW / 16, CT = C / 16, CF = C / KB;
    const LinAttnArgs& a = ca.a;
    typedef Stage<T, DKP, NT> SK;
    typedef Stage<T, DVP, NT> SV;
    __shared__ __attribute__((aligned(16))) T qs[STATE_ONLY ? 8 : C * SK::LD];
    __shared__ __attribute__((aligned(16))) T ks[C * SK::LD];
    __shared__ __attribute__((aligned(16))) T vs[C * SV::LD];
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4, v0 = (threadIdx.x >> 6) * DVW;
    const int seg = blockIdx.x % ca.nseg, bh = blockIdx.x / ca.nseg, h = bh % a.H, b = bh / a.H;
    const int n = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    const int beg = seg * ca.seg_len, end = min(n, beg + ca.seg_len);
    if (STATE_ONLY && beg + ca.seg_len >= n) return;           // no token follows: the scan does not read it
    const float g = a.g[h];
    const int e = a.rev ? 0 : 1;
    const long dir = a.rev ? -1 : 1, t0 = a.rev ? n - 1 : 0;    // position p is token t0 + dir p
    const T* q = (const T*)a.q + (long)b * a.qb + (long)(h / a.rq) * a.qh + t0 * a.qt;
    const T* k = (const T*)a.k + (long)b * a.kb + (long)(h / a.rk) * a.kh + t0 * a.kt;
    const T* v = (const T*)a.v + (long)b * a.vb + (long)(h / a.rv) * a.vh + t0 * a.vt;
    TO* o = (TO*)a.o + (long)b * a.ob + (long)h * a.oh;
    const long qt = dir * a.qt, kt = dir * a.kt, vt = dir * a.vt;

    f32x4 S[KT][VT];
    const float* s_in = STATE_ONLY ? nullptr : (seg == 0 ? a.s_in : ca.seg_state + ((long)bh * (ca.nseg - 1) + seg - 1) * a.Dk * a.Dv);
    const int si = seg == 0 ? a.si : a.Dv, sj = seg == 0 ? a.sj : 1;
    if (s_in && seg == 0) s_in += (long)bh * a.Dk * a.Dv;
    if (beg >= n && seg > 0) s_in = nullptr;                     // an empty segment: nothing is computed from it
#pragma unroll
    for (int x = 0; x < KT; ++x)
#pragma unroll
        for (int y = 0; y < VT; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 16 * x + 4 * grp + i, j = v0 + 16 * y + col;
                S[x][y][i] = (s_in && d < a.Dk && j < a.Dv) ? s_in[(long)d * si + (long)j * sj] : 0.f;
            }

    // powers of the decay: inside a tile (t - s >= 0, else nothing), one tile further (t - s + 16 >= 1), and per tile
    float pd[4], pb[4], ptile[CT], wst[CF][KB / 4], pi = 0.f;
    if constexpr (!STATE_ONLY) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = col - M::srow(grp, i);
            pd[i] = d >= 0 ? a.uscale * decay_power(g, d) : 0.f;
            pb[i] = a.uscale * decay_power(g, 16 + d);
        }
#pragma unroll
        for (int x = 0; x < CT; ++x) ptile[x] = decay_power(g, 16 * x);
        pi = decay_power(g, col + e);
    }
    auto weights = [&](int L) {
#pragma unroll
        for (int u = 0; u < CF; ++u)
#pragma unroll
            for (int j = 0; j < KB / 4; ++j) wst[u][j] = a.uscale * decay_power(g, max(0, L - e - (KB * u + 16 * (j >> 2) + M::srow(grp, j & 3))));
    };
    weights(C);
    const float em1 = expm1f(g * (float)C);

    SK rq, rk;
    SV rv;
    if (beg < end) {
        if constexpr (!STATE_ONLY) rq.load(q + beg * qt, qt, end - beg, a.Dk, ca.vq);
        rk.load(k + beg * kt, kt, end - beg, a.Dk, ca.vk);
        rv.load(v + beg * vt, vt, end - beg, a.Dv, ca.vv);
    }
    for (int c0 = beg; c0 < end; c0 += C) {
        __syncthreads();
        if constexpr (!STATE_ONLY) rq.store(qs);
        rk.store(ks);
        rv.store(vs);
        __syncthreads();
        const int L = min(C, end - c0), c1 = c0 + C;
        if (c1 < end) {
            if constexpr (!STATE_ONLY) rq.load(q + c1 * qt, qt, end - c1, a.Dk, ca.vq);
            rk.load(k + c1 * kt, kt, end - c1, a.Dk, ca.vk);
            rv.load(v + c1 * vt, vt, end - c1, a.Dv, ca.vv);
        }
        typename M::Frag vf[CF][VT];
#pragma unroll
        for (int u = 0; u < CF; ++u)
#pragma unroll
            for (int y = 0; y < VT; ++y) vf[u][y] = M::col(vs, SV::LD, v0 + 16 * y, u, lane);
        if constexpr (!STATE_ONLY) {
            f32x4 acc[CT][VT];
#pragma unroll
            for (int x = 0; x < CT; ++x)
#pragma unroll
                for (int y = 0; y < VT; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
            // q S
#pragma unroll
            for (int u = 0; u < KF; ++u) {
                typename M::Frag sf[VT][M::NS];
#pragma unroll
                for (int y = 0; y < VT; ++y) {
                    f32x4 t[TPF];
#pragma unroll
                    for (int p = 0; p < TPF; ++p) t[p] = S[u * TPF + p][y];
                    M::template pieces<M::NS>(t, sf[y]);
                }
#pragma unroll
                for (int x = 0; x < CT; ++x) {
                    const typename M::Frag qf = M::row(qs, SK::LD, 16 * x + col, u, grp);
#pragma unroll
                    for (int y = 0; y < VT; ++y)
#pragma unroll
                        for (int p = M::NS - 1; p >= 0; --p) acc[x][y] = M::mma(sf[y][p], qf, acc[x][y]);
                }
            }
#pragma unroll
            for (int x = 0; x < CT; ++x) {
                if (16 * x >= L) break;
                const float f = pi * ptile[x];
#pragma unroll
                for (int y = 0; y < VT; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[x][y][i] *= f;
                typename M::Frag qf[KF];
#pragma unroll
                for (int u = 0; u < KF; ++u) qf[u] = M::row(qs, SK::LD, 16 * x + col, u, grp);
#pragma unroll
                for (int u = 0; u < CF; ++u) {
                    if (u * TPF > x) break;
                    f32x4 t[TPF];
#pragma unroll
                    for (int p = 0; p < TPF; ++p) {
                        const int s = u * TPF + p;
                        t[p] = f32x4{0.f, 0.f, 0.f, 0.f};
                        if (s > x) continue;
#pragma unroll
                        for (int w = 0; w < KF; ++w) t[p] = M::mma(M::row(ks, SK::LD, 16 * s + M::krow(col), w, grp), qf[w], t[p]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) t[p][i] *= s == x ? pd[i] : pb[i] * ptile[x - s > 0 ? x - s - 1 : 0];
                    }
                    typename M::Frag pf[M::NS];
                    M::template pieces<M::NS>(t, pf);
#pragma unroll
                    for (int y = 0; y < VT; ++y)
#pragma unroll
                        for (int p = M::NS - 1; p >= 0; --p) acc[x][y] = M::mma(vf[u][y], pf[p], acc[x][y]);
                }
                const int r = 16 * x + col;
                if (r < L) {
                    TO* row = o + (t0 + dir * (c0 + r)) * a.ot;
#pragma unroll
                    for (int y = 0; y < VT; ++y) {
                        const int j = v0 + 16 * y + 4 * grp;
                        const float4 w = make_float4(acc[x][y][0] * a.oscale, acc[x][y][1] * a.oscale, acc[x][y][2] * a.oscale, acc[x][y][3] * a.oscale);
                        if (ca.vo) {
                            if (j < a.Dv) st4(row + j, 0, w);
                        } else {
                            if (j < a.Dv) st1(row, j, w.x);
                            if (j + 1 < a.Dv) st1(row, j + 1, w.y);
                            if (j + 2 < a.Dv) st1(row, j + 2, w.z);
                            if (j + 3 < a.Dv) st1(row, j + 3, w.w);
                        }
                    }
                }
            }
        }
        // the state
        float m1 = em1;
        if (L < C) {                                               // the last chunk of a row
            weights(L);
            m1 = expm1f(g * (float)L);
        }
#pragma unroll
        for (int x = 0; x < KT; ++x)
#pragma unroll
            for (int y = 0; y < VT; ++y)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[x][y][i] = __builtin_fmaf(S[x][y][i], m1, S[x][y][i]);
#pragma unroll
        for (int u = 0; u < CF; ++u) {
            typename M::Frag wf[VT][M::NV];
#pragma unroll
            for (int y = 0; y < VT; ++y) {
                f32x4 t[TPF];
                M::scaled(vf[u][y], wst[u], t);
                M::template pieces<M::NV>(t, wf[y]);
            }
#pragma unroll
            for (int x = 0; x < KT; ++x) {
                const typename M::Frag kf = M::col(ks, SK::LD, 16 * x, u, lane);
#pragma unroll
                for (int y = 0; y < VT; ++y)
#pragma unroll
                    for (int p = M::NV - 1; p >= 0; --p) S[x][y] = M::mma(kf, wf[y][p], S[x][y]);
            }
        }
    }
    // behind the row's last token: o is zero
    if constexpr (!STATE_ONLY) {
        const int z0 = max(n, beg), z1 = min(a.T, beg + ca.seg_len);
        for (long x = threadIdx.x; x < (long)max(0, z1 - z0) * a.Dv; x += NT) st1(o, (z0 + x / a.Dv) * a.ot + x % a.Dv, 0.f);
    }
    float* s_out = STATE_ONLY ? ca.seg_state + ((long)bh * (ca.nseg - 1) + seg) * a.Dk * a.Dv : a.s_out;
    if (!STATE_ONLY) {
        if (!s_out || seg != (n > 0 ? (n - 1) / ca.seg_len : 0)) return;      // the segment with the row's last token
        s_out += (long)bh * a.Dk * a.Dv;
    }
    const int oi = STATE_ONLY ? a.Dv : a.si, oj = STATE_ONLY ? 1 : a.sj;
#pragma unroll
    for (int x = 0; x < KT; ++x)
#pragma unroll
        for (int y = 0; y < VT; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 16 * x + 4 * grp + i, j = v0 + 16 * y + col;
                if (d < a.Dk && j < a.Dv) s_out[(long)d * oi + (long)j * oj] = S[x][y][i];
            }
}

// seg_state[i] <- the state behind segment i: one thread per element, the segments' own contributions loaded eight at a time
__global__ __launch_bounds__(256) void linattn_segment_scan_kernel(const ChunkArgs ca) {
    const LinAttnArgs& a = ca.a;
    const int x = blockIdx.y * 256 + threadIdx.x, D = a.Dk * a.Dv, bh = blockIdx.x;
    if (x >= D) return;
    const int n = a.lengths ? min(max(a.lengths[bh / a.H], 0), a.T) : a.T;
    const float g = a.g[bh % a.H];
    float* p = ca.seg_state + (long)bh * (ca.nseg - 1) * D + x;
    float run = a.s_in ? a.s_in[(long)bh * D + (long)(x / a.Dv) * a.si + (long)(x % a.Dv) * a.sj] : 0.f;
    const float em1 = expm1f(g * (float)ca.seg_len);
    for (int i0 = 0; i0 < ca.nseg - 1; i0 += 8) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (i0 + i < ca.nseg - 1 && (long)(i0 + i + 1) * ca.seg_len < n) ? p[(long)(i0 + i) * D] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i0 + i >= ca.nseg - 1 || (long)(i0 + i + 1) * ca.seg_len >= n) return;      // what follows enters no token's segment
            run = __builtin_fmaf(run, em1, run) + y[i];
            p[(long)(i0 + i) * D] = run;
        }
    }
}

// One token: a block per (batch row, head); thread = (row group, column), the partial sums over the row groups meet in LDS.
template <typename T>
__global__ __launch_bounds__(256) void linattn_step_kernel(const LinAttnArgs a) {
    __shared__ float qs[128], ks[128], red[256];
    const int h = blockIdx.x % a.H, b = blockIdx.x / a.H, tid = threadIdx.x;
    const T* q = (const T*)a.q + (long)b * a.qb + (long)(h / a.rq) * a.qh;
    const T* k = (const T*)a.k + (long)b * a.kb + (long)(h / a.rk) * a.kh;
    const T* v = (const T*)a.v + (long)b * a.vb + (long)(h / a.rv) * a.vh;
    if (tid < a.Dk) { qs[tid] = ld1(q, tid); ks[tid] = ld1(k, tid); }
    __syncthreads();
    const float lam = expf(a.g[h]);
    float* S = a.s_out + ((long)b * a.H + h) * a.Dk * a.Dv;
    const int cols = a.Dv <= 32 ? 32 : (a.Dv <= 64 ? 64 : 128), groups = 256 / cols, j = tid % cols, r0 = tid / cols;
    float acc = 0.f;
    if (j < a.Dv) {
        const float vv = ld1(v, j);
        for (int d = r0; d < a.Dk; d += groups) {
            const float s = lam * S[(long)d * a.Dv + j] + ks[d] * vv;
            S[(long)d * a.Dv + j] = s;
            acc += qs[d] * s;
        }
    }
    red[tid] = acc;
    __syncthreads();
    if (tid < a.Dv) {
        float s = 0.f;
        for (int r = 0; r < groups; ++r) s += red[r * cols + tid];
        st1((T*)a.o + (long)b * a.ob + (long)h * a.oh, tid, s * a.oscale);
    }
}

// out[r][c] = sum over j < n of x[r][c / D][j][c % D]: the gradient of a head that n heads read, in the order of the heads
template <typename T>
__global__ void head_sum_kernel(const float* __restrict__ x, T* __restrict__ out, long rows, int heads, int n, int D) {
    const long total = rows * heads * D;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const int d = (int)(i % D);
        const float* p = x + i / D * n * D + d;
        float s = p[0];
        for (int j = 1; j < n; ++j) s += p[(long)j * D];
        st1(out, i, s);
    }
}

// Segments of the time axis: one pass over q, k, v where the rows and heads alone give every compute unit a workgroup or more; otherwise the axis is
// split so that two are there, at no less than four chunks a segment, for a second read of k and v and the segments' states.
void segments(int B, int T, int H, int b16_in, int* nseg, int* len) {
    const int C = b16_in ? Mma<b16>::C : Mma<float>::C, chunks = (T + C - 1) / C, cus = hw_cu_count();
    const long rows = (long)B * H;
    long want = rows >= cus ? 1 : (2L * cus + rows - 1) / (rows > 0 ? rows : 1);
    if (want > chunks / 4) want = chunks / 4;
    if (want < 1) want = 1;
    const int per = (int)((chunks + want - 1) / want);
    *nseg = per > 0 ? (chunks + per - 1) / per : 1;
    if (*nseg < 1) *nseg = 1;
    *len = (per > 0 ? per : 1) * C;
}

template <typename T, typename TO, int DKP, int DVP> void chunk_launch(const ChunkArgs& c, hipStream_t st) {
    constexpr int NT = (DVP < 64 ? DVP / 16 : 4) * 64;
    const dim3 grid((unsigned)((long)c.a.B * c.a.H * c.nseg));
    if (c.nseg > 1) {
        hipLaunchKernelGGL((linattn_chunk_kernel<T, TO, DKP, DVP, true>), grid, dim3(NT), 0, st, c);
        hipLaunchKernelGGL(linattn_segment_scan_kernel, dim3(c.a.B * c.a.H, (c.a.Dk * c.a.Dv + 255) / 256), dim3(256), 0, st, c);
    }
    hipLaunchKernelGGL((linattn_chunk_kernel<T, TO, DKP, DVP, false>), grid, dim3(NT), 0, st, c);
}
template <typename T, typename TO, int DKP> void chunk_launch_v(const ChunkArgs& c, hipStream_t st) {
    if (c.a.Dv <= 32) chunk_launch<T, TO, DKP, 32>(c, st);
    else if (c.a.Dv <= 64) chunk_launch<T, TO, DKP, 64>(c, st);
    else chunk_launch<T, TO, DKP, 128>(c, st);
}
template <typename T, typename TO> void chunk_launch_k(const ChunkArgs& c, hipStream_t st) {
    if (c.a.Dk <= 32) chunk_launch_v<T, TO, 32>(c, st);
    else if (c.a.Dk <= 64) chunk_launch_v<T, TO, 64>(c, st);
    else chunk_launch_v<T, TO, 128>(c, st);
}

// rows of D elements are whole pieces of `bytes`, also from one row to the next
bool pieces_ok(const void* p, long b, long t, long h, int D, int elem, int bytes) {
    return (uintptr_t)p % bytes == 0 && (long)D * elem % bytes == 0 && b * elem % bytes == 0 && t * elem % bytes == 0 && h * elem % bytes == 0;
}

int fill_args(LinAttnArgs& a, const char* what, const void* q, const void* k, const void* v, void* o, const float* g, const long* strides, int B, int T,
              int H, int rq, int rk, int rv, int Dk, int Dv) {
    HA2G_REQUIRE(B >= 0 && T >= 0 && H >= 1 && Dk >= 1 && Dk <= 128 && Dv >= 1 && Dv <= 128, "%s: B=%d T=%d H=%d Dk=%d Dv=%d (1 <= Dk, Dv <= 128)", what, B,
                 T, H, Dk, Dv);
    HA2G_REQUIRE(rq >= 1 && rk >= 1 && rv >= 1 && H % rq == 0 && H % rk == 0 && H % rv == 0, "%s: %d heads shared by %d / %d / %d", what, H, rq, rk, rv);
    HA2G_REQUIRE((long)B * H <= 0x7fffffffL, "%s: B * H = %ld", what, (long)B * H);
    HA2G_REQUIRE(B == 0 || (g && (T == 0 || (q && k && v && o))), "%s: null operand", what);
    a.q = q; a.k = k; a.v = v; a.o = o; a.g = g;
    a.qb = strides[0]; a.qt = strides[1]; a.qh = strides[2]; a.kb = strides[3]; a.kt = strides[4]; a.kh = strides[5];
    a.vb = strides[6]; a.vt = strides[7]; a.vh = strides[8]; a.ob = strides[9]; a.ot = strides[10]; a.oh = strides[11];
    a.B = B; a.T = T; a.H = H; a.Dk = Dk; a.Dv = Dv; a.rq = rq; a.rk = rk; a.rv = rv;
    return 0;
}

}  // namespace

extern "C" {

long ha2g_linattn_workspace_floats(int B, int T, int H, int Dk, int Dv, int b16_in) {
    int nseg, len;
    if (B < 1 || H < 1 || T < 1) return 0;
    segments(B, T, H, b16_in, &nseg, &len);
    return (long)B * H * (nseg - 1) * Dk * Dv;
}

int ha2g_linattn(const void* q, const void* k, const void* v, void* o, const float* log_decay, const float* s_in, float* s_out, const int* lengths,
                 const long* strides, int B, int T, int H, int rq, int rk, int rv, int Dk, int Dv, int s_transposed, float o_scale, float u_scale,
                 int reverse, int b16_in, int b16_out, float* ws, void* stream) {
    ChunkArgs c;
    LinAttnArgs& a = c.a;
    if (const int rc = fill_args(a, "linattn", q, k, v, o, log_decay, strides, B, T, H, rq, rk, rv, Dk, Dv)) return rc;
    if (B == 0) return 0;
    a.s_in = s_in; a.s_out = s_out; a.lengths = lengths;
    a.si = s_transposed ? 1 : Dv; a.sj = s_transposed ? Dk : 1;
    a.oscale = o_scale; a.uscale = u_scale; a.rev = reverse;
    const hipStream_t st = (hipStream_t)stream;
    HA2G_REQUIRE(b16_in || !b16_out, "linattn: fp32 operands with a bf16 result");
    segments(B, T, H, b16_in, &c.nseg, &c.seg_len);
    HA2G_REQUIRE(c.nseg == 1 || ws, "linattn: no workspace (ha2g_linattn_workspace_floats)");
    HA2G_REQUIRE((long)B * H * c.nseg <= 0x7fffffffL, "linattn: B * H * segments = %ld", (long)B * H * c.nseg);
    HA2G_REQUIRE((long)T + c.seg_len <= 0x7fffffffL, "linattn: T = %d", T);
    c.seg_state = ws;
    const int e = b16_in ? 2 : 4, eo = b16_out ? 2 : 4;
    c.vq = pieces_ok(q, a.qb, a.qt, a.qh, Dk, e, 16);
    c.vk = pieces_ok(k, a.kb, a.kt, a.kh, Dk, e, 16);
    c.vv = pieces_ok(v, a.vb, a.vt, a.vh, Dv, e, 16);
    c.vo = pieces_ok(o, a.ob, a.ot, a.oh, Dv, eo, 4 * eo);
    if (!b16_in) chunk_launch_k<float, float>(c, st);
    else if (b16_out) chunk_launch_k<b16, b16>(c, st);
    else chunk_launch_k<b16, float>(c, st);
    HA2G_CHECK_LAUNCH("linattn");
    return 0;
}

int ha2g_linattn_step(const void* q, const void* k, const void* v, void* o, const float* log_decay, float* state, const long* strides, int B, int H,
                      int rq, int rk, int rv, int Dk, int Dv, float o_scale, int b16_io, void* stream) {
    LinAttnArgs a;
    if (const int rc = fill_args(a, "linattn_step", q, k, v, o, log_decay, strides, B, 1, H, rq, rk, rv, Dk, Dv)) return rc;
    HA2G_REQUIRE(B == 0 || state, "linattn_step: null state");
    if (B == 0) return 0;
    a.s_out = state; a.oscale = o_scale;
    if (b16_io) hipLaunchKernelGGL(linattn_step_kernel<b16>, dim3(B * H), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(linattn_step_kernel<float>, dim3(B * H), dim3(256), 0, (hipStream_t)stream, a);
    HA2G_CHECK_LAUNCH("linattn_step");
    return 0;
}

int ha2g_head_sum(const float* x, void* out, long rows, int heads, int n, int D, int b16_out, void* stream) {
    HA2G_REQUIRE(rows >= 0 && heads >= 1 && n >= 1 && D >= 1, "head_sum: rows=%ld heads=%d n=%d D=%d", rows, heads, n, D);
    if (rows == 0) return 0;
    const long total = rows * heads * D, want = (total + 255) / 256;
    const dim3 grid((unsigned)(want > 16384 ? 16384 : want));
    if (b16_out) hipLaunchKernelGGL(head_sum_kernel<b16>, grid, dim3(256), 0, (hipStream_t)stream, x, (b16*)out, rows, heads, n, D);
    else hipLaunchKernelGGL(head_sum_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, x, (float*)out, rows, heads, n, D);
    HA2G_CHECK_LAUNCH("head_sum");
    return 0;
}

}  // extern "C"
