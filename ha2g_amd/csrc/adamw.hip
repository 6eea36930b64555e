// AdamW (decoupled weight decay) over many separately allocated tensors in one launch:
//     m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2;   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in fp32 per element, the step's scalars in double by one thread that also advances t in device memory (a captured graph does so on each replay;
// two powers in double by every thread cost more than the elements).  States are fp32, or 8 bits:
// blocks of 128 consecutive elements of a tensor hold m and r = sqrt(v) as e4m3 codes times one power of two each, the smallest that brings the
// block's largest finite magnitude to at most 448.  r instead of v halves the range in octaves.  A code has 4 significant bits, so a round to
// nearest would never let v decay by its 0.1 % a step: the part below a code rounds up with its own probability, by a dither that a counter hash
// makes of (seed, t, tensor, place), the same on every run.  A root above zero keeps at least the smallest code: it divides the next update, and as
// 0 beside an m that survived (m has a scale of its own) it would let that update be lr m / eps.  Such an element's v does not decay below some 2^-36
// of its block's largest.  A value that is not finite keeps to its own element (the NaN code).
#include "common.h"

namespace {

constexpr int AW_TENSORS = 64;      // per launch: the table travels by value in the kernel's arguments
constexpr long AW_CHUNKS = (1L << 24) - 1;      // per launch: a grid has less than 2^32 threads

struct AdamWTable {
    void *p[AW_TENSORS], *g[AW_TENSORS], *m[AW_TENSORS], *v[AW_TENSORS];
    float *sm[AW_TENSORS], *sr[AW_TENSORS];
    long n[AW_TENSORS];
    int start[AW_TENSORS + 1];      // first chunk of each tensor
    int count, first;               // tensors here, number of the first one (the dither's)
    unsigned long long vec;         // bit i: tensor i's pointers allow wide accesses
};
struct AdamWScalars {
    float b1, b2, omb1, omb2, keep, eps;
    unsigned seed;
    const float* dev;               // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), t (as an integer)
    const int* guard;
};
static_assert(sizeof(AdamWTable) + sizeof(AdamWScalars) <= 4096, "kernel arguments");

__global__ void adamw_scalars_kernel(int* step, const int* guard, double lr, double b1, double b2, float* out) {
    if (guard == nullptr || *guard == 0) *step += 1;
    const double t = (double)*step;
    out[0] = (float)(lr / (1.0 - pow(b1, t)));
    out[1] = (float)(1.0 / sqrt(1.0 - pow(b2, t)));
    reinterpret_cast<int*>(out)[2] = *step;
}

__device__ __forceinline__ unsigned hash32(unsigned x) {      // factors: 2^32 over the golden ratio, and over the plastic number
    x = (x ^ (x >> 16)) * 0x9e3779b9u;
    x = (x ^ (x >> 15)) * 0xc13fa9a9u;
    return x ^ (x >> 16);
}

__device__ __forceinline__ void update(const AdamWScalars& c, float step, float root, float g, float& p, float& m, float& v, float& r) {
    m = c.b1 * m + c.omb1 * g;
    v = c.b2 * v + (c.omb2 * g) * g;
    r = sqrtf(v);
    p = p * c.keep - step * m / (r * root + c.eps);
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

// A block per chunk: long enough that its search in the table is small beside its memory time, short enough for a model's tensors to fill the chip
constexpr int CHUNK32 = 4096, CHUNK8 = 4096;

// Bound by memory: 28 bytes an element with everything in fp32.  A generator's 13.1 million parameters in 53 tensors: 57 us = 6.4 TB/s where the last
// step's data is partly in the last-level cache; 80 us = 4.6 TB/s where it is not.
template <typename TP, typename TG>
__global__ __launch_bounds__(256) void adamw32_kernel(const AdamWTable tab, const AdamWScalars sc) {
    if (sc.guard != nullptr && *sc.guard != 0) return;
    const int i = find_tensor(tab, blockIdx.x);
    const long base = (long)(blockIdx.x - tab.start[i]) * CHUNK32, n = tab.n[i];
    TP* p = (TP*)tab.p[i];
    const TG* g = (const TG*)tab.g[i];
    float *m = (float*)tab.m[i], *v = (float*)tab.v[i];
    const float step = sc.dev[0], root = sc.dev[1];
    float r;
    if ((tab.vec >> i & 1) && base + CHUNK32 <= n) {
#pragma unroll
        for (int u = 0; u < CHUNK32 / 1024; ++u) {
            const long at = (base >> 2) + u * 256 + threadIdx.x;
            float4 P = ld4(p, at), G = ld4(g, at), M = ld4(m, at), V = ld4(v, at);
            update(sc, step, root, G.x, P.x, M.x, V.x, r);
            update(sc, step, root, G.y, P.y, M.y, V.y, r);
            update(sc, step, root, G.z, P.z, M.z, V.z, r);
            update(sc, step, root, G.w, P.w, M.w, V.w, r);
            st4(p, at, P); st4(m, at, M); st4(v, at, V);
        }
        return;
    }
    const long end = min(n, base + CHUNK32);
    for (long at = base + threadIdx.x; at < end; at += 256) {
        float P = ld1(p, at), M = m[at], V = v[at];
        update(sc, step, root, ld1(g, at), P, M, V, r);
        sta(p, at, P); m[at] = M; v[at] = V;
    }
}

// |x| if it is finite, else 0
__device__ __forceinline__ float finite_abs(float x) {
    const unsigned u = __float_as_uint(x) & 0x7fffffffu;
    return __uint_as_float(u < 0x7f800000u ? u : 0u);
}
// exponent of the block's scale from its largest finite magnitude
__device__ __forceinline__ int scale_exponent(float top) {
    const unsigned u = __float_as_uint(top);
    const int field = (int)(u >> 23);
    const int e = field - 126 - 9 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (field == 0 || e < -126) ? -126 : e;
}
// a = |x| / scale <= 448 (x finite): the code of the binade, plus the 4 significant bits of a with the dither added below them
__device__ __forceinline__ unsigned encode(float x, float inv, float dither) {
    const float f = finite_abs(x), a = f * inv;
    const int ue = max((int)(__float_as_uint(a) >> 23), 121);                            // exponent field, at least that of 2^-6
    const int k = (int)(a * __uint_as_float((unsigned)(257 - ue) << 23) + dither);
    unsigned code = (unsigned)min((ue - 120) * 8 + k - 8, 126);
    code = f == fabsf(x) ? code : 0x7fu;                                                // NaN and infinities: the NaN code
    return code | (x < 0.f ? 0x80u : 0u);
}

// 16 lanes hold a block of 128 elements, 8 consecutive ones each; a thread does this for CHUNK8 / 2048 places.  Bound by memory: 14 bytes an element
// with bf16 gradients; 115 million parameters 315 us = 5.1 TB/s.
template <typename TP, typename TG>
__global__ __launch_bounds__(256) void adamw8_kernel(const AdamWTable tab, const AdamWScalars sc) {
    if (sc.guard != nullptr && *sc.guard != 0) return;
    const int i = find_tensor(tab, blockIdx.x);
    const long n = tab.n[i];
    TP* p = (TP*)tab.p[i];
    const TG* g = (const TG*)tab.g[i];
    unsigned char *mc = (unsigned char*)tab.m[i], *rc = (unsigned char*)tab.v[i];
    float *smp = tab.sm[i], *srp = tab.sr[i];
    const float step = sc.dev[0], root = sc.dev[1];
    const unsigned key = hash32(hash32(hash32(sc.seed) ^ (unsigned)__float_as_int(sc.dev[2])) ^ (unsigned)(tab.first + i));
    const bool vec = tab.vec >> i & 1;
#pragma unroll 1
    for (int u = 0; u < CHUNK8 / 2048; ++u) {
        const long at = (long)(blockIdx.x - tab.start[i]) * CHUNK8 + u * 2048 + threadIdx.x * 8;
        const bool wide = vec && at + 8 <= n, any = at < n;
        float P[8], G[8], M[8], R[8];
        unsigned cm[2] = {0u, 0u}, cr[2] = {0u, 0u};              // elements behind the end are zeros and stay zeros
        float sm = 0.f, sr = 0.f;
        if (any) { sm = smp[at >> 7]; sr = srp[at >> 7]; }
        if (wide) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 a = ld4(p, (at >> 2) + h), b = ld4(g, (at >> 2) + h);
                P[4 * h] = a.x; P[4 * h + 1] = a.y; P[4 * h + 2] = a.z; P[4 * h + 3] = a.w;
                G[4 * h] = b.x; G[4 * h + 1] = b.y; G[4 * h + 2] = b.z; G[4 * h + 3] = b.w;
            }
            const uint2 x = *reinterpret_cast<const uint2*>(mc + at), y = *reinterpret_cast<const uint2*>(rc + at);
            cm[0] = x.x; cm[1] = x.y; cr[0] = y.x; cr[1] = y.y;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                P[k] = G[k] = 0.f;
                if (at + k < n) {
                    P[k] = ld1(p, at + k);
                    G[k] = ld1(g, at + k);
                    cm[k >> 2] |= (unsigned)mc[at + k] << (8 * (k & 3));
                    cr[k >> 2] |= (unsigned)rc[at + k] << (8 * (k & 3));
                }
            }
        }
        float tm = 0.f, tr = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            M[4 * h] = __builtin_amdgcn_cvt_f32_fp8((int)cm[h], 0); M[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8((int)cm[h], 1);
            M[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8((int)cm[h], 2); M[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8((int)cm[h], 3);
            R[4 * h] = __builtin_amdgcn_cvt_f32_fp8((int)cr[h], 0); R[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8((int)cr[h], 1);
            R[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8((int)cr[h], 2); R[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8((int)cr[h], 3);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            M[k] *= sm;
            R[k] *= sr;
            float v = R[k] * R[k];
            update(sc, step, root, G[k], P[k], M[k], v, R[k]);
            tm = fmaxf(tm, finite_abs(M[k]));
            tr = fmaxf(tr, finite_abs(R[k]));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) { tm = fmaxf(tm, __shfl_xor(tm, o, 64)); tr = fmaxf(tr, __shfl_xor(tr, o, 64)); }
        const int em = scale_exponent(tm), er = scale_exponent(tr);
        const float im = __uint_as_float((unsigned)(127 - em) << 23), ir = __uint_as_float((unsigned)(127 - er) << 23);
        const unsigned place = key ^ (unsigned)(at >> 32) * 0x9e3779b9u;                  // at is a multiple of 8: its upper word is the elements'
        cm[0] = cm[1] = cr[0] = cr[1] = 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const unsigned d = hash32(((unsigned)at + k) ^ place);
            cm[k >> 2] |= encode(M[k], im, (float)(d >> 16) * 0x1p-16f) << (8 * (k & 3));
            cr[k >> 2] |= max(encode(R[k], ir, (float)(d & 0xffffu) * 0x1p-16f), R[k] > 0.f ? 1u : 0u) << (8 * (k & 3));
        }
        if (wide) {
#pragma unroll
            for (int h = 0; h < 2; ++h) st4(p, (at >> 2) + h, make_float4(P[4 * h], P[4 * h + 1], P[4 * h + 2], P[4 * h + 3]));
            *reinterpret_cast<uint2*>(mc + at) = make_uint2(cm[0], cm[1]);
            *reinterpret_cast<uint2*>(rc + at) = make_uint2(cr[0], cr[1]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (at + k < n) {
                    sta(p, at + k, P[k]);
                    mc[at + k] = (unsigned char)(cm[k >> 2] >> (8 * (k & 3)));
                    rc[at + k] = (unsigned char)(cr[k >> 2] >> (8 * (k & 3)));
                }
        }
        if (any && (threadIdx.x & 15) == 0) {
            smp[at >> 7] = __uint_as_float((unsigned)(127 + em) << 23);
            srp[at >> 7] = __uint_as_float((unsigned)(127 + er) << 23);
        }
    }
}

template <typename TP, typename TG> void adamw_launch(const AdamWTable& t, const AdamWScalars& s, int bits, hipStream_t st) {
    const dim3 grid(t.start[t.count]);
    if (bits == 32) hipLaunchKernelGGL((adamw32_kernel<TP, TG>), grid, dim3(256), 0, st, t, s);
    else hipLaunchKernelGGL((adamw8_kernel<TP, TG>), grid, dim3(256), 0, st, t, s);
}

}  // namespace

extern "C" {

int ha2g_adamw_scalars(int* step, const int* guard, double lr, double b1, double b2, float* scalars, void* stream) {
    HA2G_REQUIRE(step && scalars, "adamw_scalars: null operand");
    hipLaunchKernelGGL(adamw_scalars_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, step, guard, lr, b1, b2, scalars);
    HA2G_CHECK_LAUNCH("adamw_scalars");
    return 0;
}

// p, g, m, v (and with 8 bits sm, sr): HOST arrays of n device pointers, len: HOST array of n lengths
int ha2g_adamw_multi(int n, const long* p, const long* g, const long* m, const long* v, const long* sm, const long* sr, const long* len, int p_b16,
                     int g_b16, int bits, double lr, double b1, double b2, double eps, double wd, unsigned seed, int first, const float* scalars,
                     const int* guard, void* stream) {
    HA2G_REQUIRE(bits == 32 || bits == 8, "adamw: states of %d bits", bits);
    HA2G_REQUIRE(n >= 0 && (n == 0 || (p && g && m && v && len && scalars && (bits == 32 || (sm && sr)))), "adamw: null table");
    const AdamWScalars sc = {(float)b1, (float)b2, (float)(1.0 - b1), (float)(1.0 - b2), (float)(1.0 - lr * wd), (float)eps, seed, scalars, guard};
    const long chunk = bits == 32 ? CHUNK32 : CHUNK8;
    AdamWTable t;
    t.count = 0;
    t.vec = 0;
    t.start[0] = 0;
    auto flush = [&]() {
        if (t.count == 0 || t.start[t.count] == 0) { t.count = 0; t.vec = 0; return 0; }      // nothing, or tensors without elements
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
        HA2G_REQUIRE(chunks <= AW_CHUNKS, "adamw: tensor %d has %ld elements", i, len[i]);
        if (t.count == AW_TENSORS || (t.count && t.start[t.count] + chunks > AW_CHUNKS)) {
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
