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

// One block per (batch row, head, 64 columns of the state): a thread keeps its column in registers and walks through the tokens.
template <typename T, typename TO, int DKP>
__global__ __launch_bounds__(64) void linattn_scan_kernel(const LinAttnArgs a) {
    constexpr int TT = 16;
    __shared__ float qs[TT][DKP], ks[TT][DKP];
    const int h = blockIdx.x % a.H, b = blockIdx.x / a.H, j = blockIdx.y * 64 + threadIdx.x;
    const bool col = j < a.Dv;
    const int n = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    const float lam = expf(a.g[h]);
    const T* q = (const T*)a.q + (long)b * a.qb + (long)(h / a.rq) * a.qh;
    const T* k = (const T*)a.k + (long)b * a.kb + (long)(h / a.rk) * a.kh;
    const T* v = (const T*)a.v + (long)b * a.vb + (long)(h / a.rv) * a.vh;
    TO* o = (TO*)a.o + (long)b * a.ob + (long)h * a.oh;
    const long sbase = ((long)b * a.H + h) * a.Dk * a.Dv;
    float S[DKP];
#pragma unroll
    for (int d = 0; d < DKP; ++d) S[d] = (a.s_in && col && d < a.Dk) ? a.s_in[sbase + (long)d * a.si + (long)j * a.sj] : 0.f;
    for (int t0 = 0; t0 < n; t0 += TT) {
        const int m = min(TT, n - t0);
        __syncthreads();
        for (int i = threadIdx.x; i < TT * DKP; i += 64) {
            const int r = i / DKP, d = i % DKP;
            const long t = a.rev ? n - 1 - (t0 + r) : t0 + r;
            const bool in = r < m && d < a.Dk;
            qs[r][d] = in ? ld1(q, t * a.qt + d) : 0.f;
            ks[r][d] = in ? ld1(k, t * a.kt + d) * a.uscale : 0.f;
        }
        __syncthreads();
        for (int r = 0; r < m; ++r) {
            const long t = a.rev ? n - 1 - (t0 + r) : t0 + r;
            const float vv = col ? ld1(v, t * a.vt + j) : 0.f;
            float acc = 0.f;
#pragma unroll
            for (int d = 0; d < DKP; ++d) {
                const float s = (a.rev ? S[d] : lam * S[d]) + ks[r][d] * vv;
                acc += qs[r][d] * s;
                S[d] = a.rev ? lam * s : s;
            }
            if (col) st1(o, t * a.ot + j, acc * a.oscale);
        }
    }
    if (col) {
        for (int t = n; t < a.T; ++t) st1(o, (long)t * a.ot + j, 0.f);
        if (a.s_out)
#pragma unroll
            for (int d = 0; d < DKP; ++d)
                if (d < a.Dk) a.s_out[sbase + (long)d * a.si + (long)j * a.sj] = S[d];
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

template <typename T, typename TO>
void scan_launch(const LinAttnArgs& a, hipStream_t st) {
    const dim3 grid(a.B * a.H, (a.Dv + 63) / 64);
    if (a.Dk <= 32) hipLaunchKernelGGL((linattn_scan_kernel<T, TO, 32>), grid, dim3(64), 0, st, a);
    else if (a.Dk <= 64) hipLaunchKernelGGL((linattn_scan_kernel<T, TO, 64>), grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL((linattn_scan_kernel<T, TO, 128>), grid, dim3(64), 0, st, a);
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

int ha2g_linattn(const void* q, const void* k, const void* v, void* o, const float* log_decay, const float* s_in, float* s_out, const int* lengths,
                 const long* strides, int B, int T, int H, int rq, int rk, int rv, int Dk, int Dv, int s_transposed, float o_scale, float u_scale,
                 int reverse, int b16_in, int b16_out, void* stream) {
    LinAttnArgs a;
    if (const int rc = fill_args(a, "linattn", q, k, v, o, log_decay, strides, B, T, H, rq, rk, rv, Dk, Dv)) return rc;
    if (B == 0) return 0;
    a.s_in = s_in; a.s_out = s_out; a.lengths = lengths;
    a.si = s_transposed ? 1 : Dv; a.sj = s_transposed ? Dk : 1;
    a.oscale = o_scale; a.uscale = u_scale; a.rev = reverse;
    const hipStream_t st = (hipStream_t)stream;
    HA2G_REQUIRE(b16_in || !b16_out, "linattn: fp32 operands with a bf16 result");
    if (!b16_in) scan_launch<float, float>(a, st);
    else if (b16_out) scan_launch<b16, b16>(a, st);
    else scan_launch<b16, float>(a, st);
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
