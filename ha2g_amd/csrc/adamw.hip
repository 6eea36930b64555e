// AdamW (decoupled weight decay) over many separately allocated tensors in one launch:
//     m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2;   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in fp32 per element, the step's scalars in double, t read from device memory (a captured graph advances it).  States are fp32, or 8 bits:
// blocks of 128 consecutive elements of a tensor hold m and r = sqrt(v) as e4m3 codes times one power of two each, the smallest that brings the
// block's largest finite magnitude to at most 448.  r instead of v halves the range in octaves.  A code has 4 significant bits, so a round to
// nearest would never let v decay by its 0.1 % a step: the part below a code rounds up with its own probability, by a dither that a counter hash
// makes of (seed, t, tensor, place), the same on every run.  A value that is not finite keeps to its own element (the NaN code).
#include "common.h"

namespace {

constexpr int AW_TENSORS = 48;      // per launch: the table travels by value in the kernel's arguments (48 * 60 bytes of the 4 KB)

struct AdamWTable {
    void *p[AW_TENSORS], *g[AW_TENSORS], *m[AW_TENSORS], *v[AW_TENSORS];
    float *sm[AW_TENSORS], *sr[AW_TENSORS];
    long n[AW_TENSORS];
    int start[AW_TENSORS + 1];      // first chunk of each tensor
    int count, first;               // tensors here, number of the first one (the dither's)
    unsigned long long vec;         // bit i: tensor i's pointers allow wide accesses
};

struct AdamWScalars {
    double lr, b1, b2, eps, wd;
    unsigned seed;
    const int *step, *guard;
};

__device__ __forceinline__ unsigned hash32(unsigned x) {      // factors: 2^32 over the golden ratio, and over the plastic number
    x = (x ^ (x >> 16)) * 0x9e3779b9u;
    x = (x ^ (x >> 15)) * 0xc13fa9a9u;
    return x ^ (x >> 16);
}

struct StepScalars { float b1, b2, omb1, omb2, keep, step, root, eps; };
__device__ __forceinline__ StepScalars step_scalars(const AdamWScalars& s) {
    const double t = (double)*s.step;
    return {(float)s.b1, (float)s.b2, (float)(1.0 - s.b1), (float)(1.0 - s.b2), (float)(1.0 - s.lr * s.wd), (float)(s.lr / (1.0 - pow(s.b1, t))),
            (float)(1.0 / sqrt(1.0 - pow(s.b2, t))), (float)s.eps};
}
__device__ __forceinline__ void update(const StepScalars& c, float g, float& p, float& m, float& v) {
    m = c.b1 * m + c.omb1 * g;
    v = c.b2 * v + (c.omb2 * g) * g;
    p = p * c.keep - c.step * m / (sqrtf(v) * c.root + c.eps);
}
__device__ __forceinline__ void sta(float* p, long i, float x) { p[i] = x; }
__device__ __forceinline__ void sta(b16* p, long i, float x) { unsigned h, l; split2_bf16(x, 0.f, h, l); p[i] = (b16)(h & 0xffff); }

// the tensor that chunk `c` lies in (uniform over the block)
__device__ __forceinline__ int find_tensor(const AdamWTable& t, int c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.start[mid] <= c) lo = mid; else hi = mid - 1;
    }
    return lo;
}

constexpr int CHUNK32 = 4096, CHUNK8 = 2048;

template <typename TP, typename TG>
__global__ __launch_bounds__(256) void adamw32_kernel(const AdamWTable tab, const AdamWScalars sc) {
    if (sc.guard != nullptr && *sc.guard != 0) return;
    const int i = find_tensor(tab, blockIdx.x);
    const long base = (long)(blockIdx.x - tab.start[i]) * CHUNK32, n = tab.n[i];
    TP* p = (TP*)tab.p[i];
    const TG* g = (const TG*)tab.g[i];
    float *m = (float*)tab.m[i], *v = (float*)tab.v[i];
    const StepScalars c = step_scalars(sc);
    if ((tab.vec >> i & 1) && base + CHUNK32 <= n) {
#pragma unroll
        for (int u = 0; u < CHUNK32 / 1024; ++u) {
            const long at = (base >> 2) + u * 256 + threadIdx.x;
            float4 P = ld4(p, at), G = ld4(g, at), M = ld4(m, at), V = ld4(v, at);
            update(c, G.x, P.x, M.x, V.x);
            update(c, G.y, P.y, M.y, V.y);
            update(c, G.z, P.z, M.z, V.z);
            update(c, G.w, P.w, M.w, V.w);
            st4(p, at, P); st4(m, at, M); st4(v, at, V);
        }
        return;
    }
    const long end = min(n, base + CHUNK32);
    for (long at = base + threadIdx.x; at < end; at += 256) {
        float P = ld1(p, at), M = m[at], V = v[at];
        update(c, ld1(g, at), P, M, V);
        sta(p, at, P); m[at] = M; v[at] = V;
    }
}

__device__ __forceinline__ float code_value(unsigned code) {                   // one e4m3 code
    return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
}
__device__ __forceinline__ bool finite_f(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
// exponent of the block's scale from its largest finite magnitude
__device__ __forceinline__ int scale_exponent(float top) {
    const unsigned u = __float_as_uint(top);
    const int field = (int)(u >> 23);
    const int e = field - 126 - 9 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (field == 0 || e < -126) ? -126 : e;
}
__device__ __forceinline__ unsigned encode(float x, float inv, unsigned dither) {
    if (!finite_f(x)) return 0x7f;
    const float a = fabsf(x) * inv;
    int ue = (int)(__float_as_uint(a) >> 23) - 127;
    if (ue < -6) ue = -6;
    const int k = (int)(a * __uint_as_float((unsigned)(130 - ue) << 23) + (float)dither * 0x1p-16f);
    const int code = (ue + 7) * 8 + k - 8;
    return (unsigned)(code > 126 ? 126 : code) | (x < 0.f ? 0x80u : 0u);
}

// 16 lanes hold a block of 128 elements, 8 consecutive ones each
template <typename TP, typename TG>
__global__ __launch_bounds__(256) void adamw8_kernel(const AdamWTable tab, const AdamWScalars sc) {
    if (sc.guard != nullptr && *sc.guard != 0) return;
    const int i = find_tensor(tab, blockIdx.x);
    const long at = (long)(blockIdx.x - tab.start[i]) * CHUNK8 + threadIdx.x * 8, n = tab.n[i];
    TP* p = (TP*)tab.p[i];
    const TG* g = (const TG*)tab.g[i];
    unsigned char *mc = (unsigned char*)tab.m[i], *rc = (unsigned char*)tab.v[i];
    const StepScalars c = step_scalars(sc);
    const bool wide = (tab.vec >> i & 1) && at + 8 <= n, any = at < n;
    float P[8], G[8], M[8], R[8];
    unsigned char cm[8] = {0}, cr[8] = {0};
    float sm = 0.f, sr = 0.f;
    if (any) { sm = tab.sm[i][at >> 7]; sr = tab.sr[i][at >> 7]; }
    if (wide) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float4 a = ld4(p, (at >> 2) + h), b = ld4(g, (at >> 2) + h);
            P[4 * h] = a.x; P[4 * h + 1] = a.y; P[4 * h + 2] = a.z; P[4 * h + 3] = a.w;
            G[4 * h] = b.x; G[4 * h + 1] = b.y; G[4 * h + 2] = b.z; G[4 * h + 3] = b.w;
        }
        *reinterpret_cast<uint2*>(cm) = *reinterpret_cast<const uint2*>(mc + at);
        *reinterpret_cast<uint2*>(cr) = *reinterpret_cast<const uint2*>(rc + at);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool in = at + k < n;
            P[k] = in ? ld1(p, at + k) : 0.f;
            G[k] = in ? ld1(g, at + k) : 0.f;
            if (in) { cm[k] = mc[at + k]; cr[k] = rc[at + k]; }
        }
    }
    float tm = 0.f, tr = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float r = code_value(cr[k]) * sr;
        float v = r * r;
        M[k] = code_value(cm[k]) * sm;
        update(c, G[k], P[k], M[k], v);
        R[k] = sqrtf(v);
        if (at + k >= n) M[k] = R[k] = 0.f;
        if (finite_f(M[k])) tm = fmaxf(tm, fabsf(M[k]));
        if (finite_f(R[k])) tr = fmaxf(tr, R[k]);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) { tm = fmaxf(tm, __shfl_xor(tm, o, 64)); tr = fmaxf(tr, __shfl_xor(tr, o, 64)); }
    const int em = scale_exponent(tm), er = scale_exponent(tr);
    const float im = __uint_as_float((unsigned)(127 - em) << 23), ir = __uint_as_float((unsigned)(127 - er) << 23);
    const unsigned key = hash32(hash32(hash32(sc.seed) ^ (unsigned)*sc.step) ^ (unsigned)(tab.first + i));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const unsigned long long e = (unsigned long long)(at + k);
        const unsigned d = hash32((unsigned)e ^ (unsigned)(e >> 32) * 0x9e3779b9u ^ key);
        cm[k] = (unsigned char)encode(M[k], im, d >> 16);
        cr[k] = (unsigned char)encode(R[k], ir, d & 0xffff);
    }
    if (wide) {
#pragma unroll
        for (int h = 0; h < 2; ++h) st4(p, (at >> 2) + h, make_float4(P[4 * h], P[4 * h + 1], P[4 * h + 2], P[4 * h + 3]));
        *reinterpret_cast<uint2*>(mc + at) = *reinterpret_cast<const uint2*>(cm);
        *reinterpret_cast<uint2*>(rc + at) = *reinterpret_cast<const uint2*>(cr);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (at + k < n) { sta(p, at + k, P[k]); mc[at + k] = cm[k]; rc[at + k] = cr[k]; }
    }
    if (any && (threadIdx.x & 15) == 0) {
        tab.sm[i][at >> 7] = __uint_as_float((unsigned)(127 + em) << 23);
        tab.sr[i][at >> 7] = __uint_as_float((unsigned)(127 + er) << 23);
    }
}

template <typename TP, typename TG> void adamw_launch(const AdamWTable& t, const AdamWScalars& s, int bits, hipStream_t st) {
    const dim3 grid(t.start[t.count]);
    if (bits == 32) hipLaunchKernelGGL((adamw32_kernel<TP, TG>), grid, dim3(256), 0, st, t, s);
    else hipLaunchKernelGGL((adamw8_kernel<TP, TG>), grid, dim3(256), 0, st, t, s);
}

}  // namespace

extern "C" {

// p, g, m, v (and with 8 bits sm, sr): HOST arrays of n device pointers, len: HOST array of n lengths
int ha2g_adamw_multi(int n, const long* p, const long* g, const long* m, const long* v, const long* sm, const long* sr, const long* len, int p_b16,
                     int g_b16, int bits, double lr, double b1, double b2, double eps, double wd, unsigned seed, int first, const int* step,
                     const int* guard, void* stream) {
    HA2G_REQUIRE(bits == 32 || bits == 8, "adamw: states of %d bits", bits);
    HA2G_REQUIRE(n >= 0 && (n == 0 || (p && g && m && v && len && step && (bits == 32 || (sm && sr)))), "adamw: null table");
    const AdamWScalars sc = {lr, b1, b2, eps, wd, seed, step, guard};
    const long chunk = bits == 32 ? CHUNK32 : CHUNK8;
    AdamWTable t;
    t.count = 0;
    t.vec = 0;
    t.start[0] = 0;
    auto flush = [&]() {
        if (t.count == 0) return 0;
        const hipStream_t st = (hipStream_t)stream;
        if (p_b16) { if (g_b16) adamw_launch<b16, b16>(t, sc, bits, st); else adamw_launch<b16, float>(t, sc, bits, st); }
        else { if (g_b16) adamw_launch<float, b16>(t, sc, bits, st); else adamw_launch<float, float>(t, sc, bits, st); }
        t.count = 0;
        t.vec = 0;
        HA2G_CHECK_LAUNCH("adamw");
        return 0;
    };
    for (int i = 0; i < n; ++i) {
        HA2G_REQUIRE(len[i] >= 0, "adamw: tensor %d has %ld elements", i, len[i]);
        const long chunks = (len[i] + chunk - 1) / chunk;
        HA2G_REQUIRE(chunks <= 0x7fffffffL / 2, "adamw: tensor %d has %ld elements", i, len[i]);
        if (t.count == AW_TENSORS || (t.count && t.start[t.count] + chunks > 0x7fffffffL)) {
            if (const int rc = flush()) return rc;
        }
        if (t.count == 0) t.first = first + i;
        HA2G_REQUIRE(len[i] == 0 || (p[i] && g[i] && m[i] && v[i] && (bits == 32 || (sm[i] && sr[i]))), "adamw: tensor %d is null", i);
        const int k = t.count++;
        t.p[k] = (void*)p[i]; t.g[k] = (void*)g[i]; t.m[k] = (void*)m[i]; t.v[k] = (void*)v[i];
        t.sm[k] = bits == 8 ? (float*)sm[i] : nullptr;
        t.sr[k] = bits == 8 ? (float*)sr[i] : nullptr;
        t.n[k] = len[i];
        t.start[k + 1] = (t.start[k] = k ? t.start[k] : 0) + (int)chunks;
        const long pa = p_b16 ? 8 : 16, ga = g_b16 ? 8 : 16, sa = bits == 32 ? 16 : 8;
        if (p[i] % pa == 0 && g[i] % ga == 0 && m[i] % sa == 0 && v[i] % sa == 0) t.vec |= 1ull << k;
    }
    return flush();
}

}  // extern "C"
