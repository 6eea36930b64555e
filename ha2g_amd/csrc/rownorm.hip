// Row norms and the tail of a block, forward and backward.  A row of C values is normalised in G groups of C / G (all of it, or per head):
//     RMS:   x^ = x / sqrt(mean(x^2) + eps)          layer:  x^ = (x - mean(x)) / sqrt(mean((x - mean)^2) + eps)
//     n = x^ w + b;   u = n act(gate);   h = alpha res + s u;   z = norm(h) w2 + b2   (over the whole row)
// Everything behind `n` is optional.  Statistics, products and sums are fp32 (the columns' sums over the rows end in double); h, z and the
// gradients are rounded once where they are stored, and z is the norm of h BEFORE that rounding, in the backward pass as in the forward one
// (h is formed again from y, res and gate there: the same bytes as reading h, and the parameters' gradients stay fp32-exact).
// Bound by HBM: a row lives in the registers of TPR threads (NI chunks of VEC values each) between its one read and its one write.
#include "common.h"

namespace {

struct TailArgs {
    const void *y, *res, *gate;
    const float *w, *b, *s, *w2, *b2;
    void *h, *z;
    float *mu, *rs, *mu2, *rs2;      // [rows * G] and [rows], kept for the backward pass (forward: nullptr = not kept; mu, mu2 for `layer` only)
    // backward
    const void *dh, *dz;
    void *dy, *dres, *dgate;
    float *part;                     // [blocks][nvec][C] sums over a block's rows: w, b, then s, then w2, b2
    float *gpart;                    // [outer][slices][C] sums of the gate's gradient over the slice's rows (gate shared by a sequence's rows)
    long inner;                      // rows of a sequence (= all rows where the gate is per row)
    int outer, C, G, layer, act, gate_shared;
    float alpha, eps;
};

template <int VEC> __device__ __forceinline__ void load_row(const float* p, long at, float* x) {
    if constexpr (VEC == 4) { const float4 v = *reinterpret_cast<const float4*>(p + at); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
    else x[0] = p[at];
}
template <int VEC> __device__ __forceinline__ void load_row(const b16* p, long at, float* x) {
    if constexpr (VEC == 4) { const float4 v = ld4(p + at, 0); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
    else x[0] = ld1(p, at);
}
template <int VEC> __device__ __forceinline__ void store_row(float* p, long at, const float* x) {
    if constexpr (VEC == 4) *reinterpret_cast<float4*>(p + at) = make_float4(x[0], x[1], x[2], x[3]);
    else p[at] = x[0];
}
template <int VEC> __device__ __forceinline__ void store_row(b16* p, long at, const float* x) {
    if constexpr (VEC == 4) st4(p + at, 0, make_float4(x[0], x[1], x[2], x[3]));
    else { unsigned h, l; split2_bf16(x[0], 0.f, h, l); p[at] = (b16)(h & 0xffff); }
}

// the gate's activation and its derivative
__device__ __forceinline__ float gate_act(float g, int act) { return act == 0 ? g : (act == 3 ? sigmoidf_(g) : g * sigmoidf_(g)); }
__device__ __forceinline__ float gate_act_d(float g, int act) {
    if (act == 0) return 1.f;
    const float s = sigmoidf_(g);
    return act == 3 ? s * (1.f - s) : s * (1.f + g * (1.f - s));
}

// Sums over the row's TPR threads of one value per chunk: r[i] = the sum over the group chunk i belongs to.  One group: a butterfly (and, for more
// than a wave, LDS).  Several: every chunk's value goes to LDS, 16 lanes add up a group, its sum is read back from the group's first place.
// Every thread of the block calls it the same number of times.
template <int TPR, int NI> struct RowSum {
    float* lds;                  // this row's TPR * NI floats
    int lane, G, cpg, nch;       // thread of the row, groups, chunks per group, chunks
    __device__ __forceinline__ float all(float s) {
        s = wave_sum(s);
        if constexpr (TPR > 64) {
            __syncthreads();
            if ((lane & 63) == 0) lds[lane >> 6] = s;
            __syncthreads();
            s = 0.f;
#pragma unroll
            for (int i = 0; i < TPR / 64; ++i) s += lds[i];
        }
        return s;
    }
    __device__ __forceinline__ void groups(const float (&p)[NI], float (&r)[NI]) {
        if (G == 1) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NI; ++i) s += p[i];
            s = all(s);
#pragma unroll
            for (int i = 0; i < NI; ++i) r[i] = s;
            return;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            if (c < nch) lds[c] = p[i];
        }
        __syncthreads();
        for (int g = lane >> 4; g < G; g += TPR / 16) {
            float s = 0.f;
            for (int c = lane & 15; c < cpg; c += 16) s += lds[g * cpg + c];
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
            if ((lane & 15) == 0) lds[g * cpg] = s;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            r[i] = c < nch ? lds[c / cpg * cpg] : 0.f;
        }
    }
};

// x -> x^ in place; r / m: 1 / std and mean per chunk
template <int TPR, int NI, int VEC>
__device__ __forceinline__ void normalise(RowSum<TPR, NI>& rsum, float (&x)[NI][VEC], float (&m)[NI], float (&r)[NI], bool layer, float inv, float eps) {
    float p[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) m[i] = 0.f;
    if (layer) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            p[i] = 0.f;
#pragma unroll
            for (int j = 0; j < VEC; ++j) p[i] += x[i][j];
        }
        rsum.groups(p, m);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            m[i] *= inv;
            const bool in = rsum.lane + i * TPR < rsum.nch;
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[i][j] = in ? x[i][j] - m[i] : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        p[i] = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p[i] += x[i][j] * x[i][j];
    }
    rsum.groups(p, r);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        r[i] = 1.0f / sqrtf(r[i] * inv + eps);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[i][j] *= r[i];
    }
}

template <int TPR> constexpr int block_of() { return TPR > 256 ? TPR : 256; }

template <typename T, int TPR, int NI, int VEC>
__global__ __launch_bounds__(block_of<TPR>()) void tail_fwd_kernel(const TailArgs a) {
    constexpr int RPB = block_of<TPR>() / TPR;
    __shared__ float lds[RPB * TPR * NI];
    const int sub = threadIdx.x / TPR, lane = threadIdx.x % TPR, nch = a.C / VEC;
    const long rows = a.inner * a.outer;
    RowSum<TPR, NI> gsum{lds + sub * TPR * NI, lane, a.G, nch / a.G, nch}, rsum{lds + sub * TPR * NI, lane, 1, nch, nch};
    for (long r0 = (long)blockIdx.x * RPB; r0 < rows; r0 += (long)gridDim.x * RPB) {
        const long row = r0 + sub;
        const bool in = row < rows;
        const long at = row * a.C, gat = a.gate_shared ? row / a.inner * a.C : at;
        float x[NI][VEC], m[NI], r[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[i][j] = 0.f;
            if (in && c < nch) load_row<VEC>((const T*)a.y, at + (long)c * VEC, x[i]);
        }
        if (a.w) {
            normalise<TPR, NI, VEC>(gsum, x, m, r, a.layer, (float)a.G / a.C, a.eps);
            if (a.rs && in) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int c = lane + i * TPR, g = c / gsum.cpg;
                    if (c < nch && c == g * gsum.cpg) {
                        a.rs[row * a.G + g] = r[i];
                        if (a.layer) a.mu[row * a.G + g] = m[i];
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            if (!(in && c < nch)) continue;
            float t[VEC];
            if (a.w) {
                load_row<VEC>(a.w, (long)c * VEC, t);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][j] *= t[j];
            }
            if (a.b) {
                load_row<VEC>(a.b, (long)c * VEC, t);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][j] += t[j];
            }
            if (a.gate) {
                load_row<VEC>((const T*)a.gate, gat + (long)c * VEC, t);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][j] *= gate_act(t[j], a.act);
            }
            if (a.s) {
                load_row<VEC>(a.s, (long)c * VEC, t);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][j] *= t[j];
            }
            if (a.res) {
                load_row<VEC>((const T*)a.res, at + (long)c * VEC, t);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][j] = a.alpha * t[j] + x[i][j];
            }
            store_row<VEC>((T*)a.h, at + (long)c * VEC, x[i]);
        }
        if (a.w2) {
            normalise<TPR, NI, VEC>(rsum, x, m, r, a.layer, 1.0f / a.C, a.eps);
            if (a.rs2 && in && lane == 0) {
                a.rs2[row] = r[0];
                if (a.layer) a.mu2[row] = m[0];
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = lane + i * TPR;
                if (!(in && c < nch)) continue;
                float t[VEC];
                load_row<VEC>(a.w2, (long)c * VEC, t);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][j] *= t[j];
                if (a.b2) {
                    load_row<VEC>(a.b2, (long)c * VEC, t);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) x[i][j] += t[j];
                }
                store_row<VEC>((T*)a.z, at + (long)c * VEC, x[i]);
            }
        }
    }
}

// A block walks through the rows of its slice of a sequence and keeps the columns' sums in registers; its partial sums leave it once.
// FULL: with gate, scale, residual or second norm; otherwise the norm alone (w, b).
template <typename T, int TPR, int NI, int VEC, bool FULL>
__global__ __launch_bounds__(block_of<TPR>()) void tail_bwd_kernel(const TailArgs a) {
    constexpr int RPB = block_of<TPR>() / TPR, NV = FULL ? 6 : 2;      // w, b, s, w2, b2, gate
    __shared__ float lds[RPB * TPR * NI * (VEC > 1 && RPB > 1 ? VEC : 1)];
    const int sub = threadIdx.x / TPR, lane = threadIdx.x % TPR, nch = a.C / VEC;
    float* const mine = lds + sub * TPR * NI;
    RowSum<TPR, NI> gsum{mine, lane, a.G, nch / a.G, nch}, rsum{mine, lane, 1, nch, nch};
    const long per = (a.inner + gridDim.x - 1) / gridDim.x, beg = blockIdx.x * per, end = min(a.inner, beg + per);
    const float inv = (float)a.G / a.C, inv2 = 1.0f / a.C;
    float acc[NV][NI][VEC];
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[n][i][j] = 0.f;
    for (long q0 = beg; q0 < end; q0 += RPB) {
        const bool in = q0 + sub < end;
        const long row = (long)blockIdx.y * a.inner + q0 + sub;
        const long at = row * a.C, gat = a.gate_shared ? (long)blockIdx.y * a.C : at;
        float y[NI][VEC], d[NI][VEC], r[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            r[i] = 0.f;
#pragma unroll
            for (int j = 0; j < VEC; ++j) y[i][j] = d[i][j] = 0.f;
            if (!(in && c < nch)) continue;
            load_row<VEC>((const T*)a.y, at + (long)c * VEC, y[i]);
            if (a.dh) load_row<VEC>((const T*)a.dh, at + (long)c * VEC, d[i]);
            if (a.w) {
                const long g = row * a.G + c / gsum.cpg;
                const float m = a.layer ? a.mu[g] : 0.f;
                r[i] = a.rs[g];
#pragma unroll
                for (int j = 0; j < VEC; ++j) y[i][j] = (y[i][j] - m) * r[i];
            }
        }
        // y = x^ (or x without a norm), d = dh
        if constexpr (FULL) {
            if (a.w2) {
                float hh[NI][VEC], e[NI][VEC], s1 = 0.f, s2 = 0.f;
                const float m2 = (in && a.layer) ? a.mu2[row] : 0.f, r2 = in ? a.rs2[row] : 0.f;
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int c = lane + i * TPR;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) hh[i][j] = e[i][j] = 0.f;
                    if (!(in && c < nch)) continue;
                    float t[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) hh[i][j] = y[i][j];
                    if (a.w) {
                        load_row<VEC>(a.w, (long)c * VEC, t);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) hh[i][j] *= t[j];
                    }
                    if (a.b) {
                        load_row<VEC>(a.b, (long)c * VEC, t);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) hh[i][j] += t[j];
                    }
                    if (a.gate) {
                        load_row<VEC>((const T*)a.gate, gat + (long)c * VEC, t);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) hh[i][j] *= gate_act(t[j], a.act);
                    }
                    if (a.s) {
                        load_row<VEC>(a.s, (long)c * VEC, t);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) hh[i][j] *= t[j];
                    }
                    if (a.res) {
                        load_row<VEC>((const T*)a.res, at + (long)c * VEC, t);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) hh[i][j] = a.alpha * t[j] + hh[i][j];
                    }
                    if (a.dz) load_row<VEC>((const T*)a.dz, at + (long)c * VEC, e[i]);
                    load_row<VEC>(a.w2, (long)c * VEC, t);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        hh[i][j] = (hh[i][j] - m2) * r2;
                        acc[3][i][j] += e[i][j] * hh[i][j];
                        acc[4][i][j] += e[i][j];
                        e[i][j] *= t[j];
                        s1 += e[i][j] * hh[i][j];
                        s2 += e[i][j];
                    }
                }
                s1 = rsum.all(s1) * inv2;
                s2 = a.layer ? rsum.all(s2) * inv2 : 0.f;
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) d[i][j] += r2 * (e[i][j] - hh[i][j] * s1 - s2);
            }
        }
        // d = the whole gradient of h (of n, where there is nothing behind it) -> d(x^)
        float p1[NI], p2[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            p1[i] = p2[i] = 0.f;
            if (!(in && c < nch)) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[i][j] = 0.f;
                continue;
            }
            float w[VEC], t[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) w[j] = 1.f;
            if (a.w) load_row<VEC>(a.w, (long)c * VEC, w);
            if constexpr (FULL) {
                float n[VEC], gt[VEC], ga[VEC];
                if (a.dres) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) t[j] = a.alpha * d[i][j];
                    store_row<VEC>((T*)a.dres, at + (long)c * VEC, t);
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) { n[j] = y[i][j] * w[j]; ga[j] = 1.f; }
                if (a.b) {
                    load_row<VEC>(a.b, (long)c * VEC, t);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) n[j] += t[j];
                }
                if (a.gate) {
                    load_row<VEC>((const T*)a.gate, gat + (long)c * VEC, gt);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) ga[j] = gate_act(gt[j], a.act);
                }
                if (a.s) {
                    load_row<VEC>(a.s, (long)c * VEC, t);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) { acc[2][i][j] += d[i][j] * (n[j] * ga[j]); d[i][j] *= t[j]; }
                }
                if (a.gate) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        t[j] = d[i][j] * n[j] * gate_act_d(gt[j], a.act);
                        acc[5][i][j] += t[j];
                        d[i][j] *= ga[j];
                    }
                    if (a.dgate && !a.gate_shared) store_row<VEC>((T*)a.dgate, at + (long)c * VEC, t);
                }
            }
            if (a.w) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    acc[0][i][j] += d[i][j] * y[i][j];
                    acc[1][i][j] += d[i][j];
                    d[i][j] *= w[j];
                    p1[i] += d[i][j] * y[i][j];
                    p2[i] += d[i][j];
                }
            }
        }
        if (a.w) {
            float c1[NI], c2[NI];
            gsum.groups(p1, c1);
            if (a.layer) gsum.groups(p2, c2);
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[i][j] = r[i] * (d[i][j] - y[i][j] * (c1[i] * inv) - (a.layer ? c2[i] * inv : 0.f));
        }
        if (a.dy) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = lane + i * TPR;
                if (in && c < nch) store_row<VEC>((T*)a.dy, at + (long)c * VEC, d[i]);
            }
        }
    }
    const bool have[6] = {a.w != nullptr, a.w != nullptr, a.s != nullptr, a.w2 != nullptr, a.w2 != nullptr, a.gate_shared && a.gpart};
    int nvec = 0, k = 0;
#pragma unroll
    for (int n = 0; n < 5; ++n) nvec += have[n];
    const long blk = (long)blockIdx.y * gridDim.x + blockIdx.x;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        if (!have[n]) continue;
        float* out = n == 5 ? a.gpart + blk * a.C : a.part + (blk * nvec + k) * a.C;
        ++k;
        if constexpr (RPB > 1) {                     // the block's rows in turn: the sums of its RPB rows meet in LDS, in the order of the rows
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = lane + i * TPR;
                if (c < nch)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) lds[(sub * NI * TPR + c) * VEC + j] = acc[n][i][j];
            }
            __syncthreads();
            for (int c = threadIdx.x; c < a.C; c += RPB * TPR) {
                float s = 0.f;
#pragma unroll
                for (int q = 0; q < RPB; ++q) s += lds[q * NI * TPR * VEC + c];
                out[c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = lane + i * TPR;
                if (c < nch) store_row<VEC>(out, (long)c * VEC, acc[n][i]);
            }
        }
    }
}

// out[o][c] = sum over p of x[o][p][c], p in ascending order within each of 16 interleaved runs, in double
template <typename T>
__global__ __launch_bounds__(1024) void slab_sum_kernel(const float* __restrict__ x, T* __restrict__ out, int n, int C) {
    __shared__ double sh[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    const float* p = x + (long)blockIdx.y * n * C + c;
    double s = 0.0;
    if (c < C) {
        int i = w;
        for (; i + 48 < n; i += 64) {
            const float v0 = p[(long)i * C], v1 = p[(long)(i + 16) * C], v2 = p[(long)(i + 32) * C], v3 = p[(long)(i + 48) * C];
            s += (double)v0; s += (double)v1; s += (double)v2; s += (double)v3;
        }
        for (; i < n; i += 16) s += (double)p[(long)i * C];
    }
    sh[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < C) {
        s = 0.0;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += sh[i][lane];
        float f = (float)s;
        store_row<1>(out, (long)blockIdx.y * C + c, &f);
    }
}

// threads per row and chunks per thread: a wave holds up to 1 024 values (256 one by one), 256 threads up to 4 096, a block of 1 024 the rest
#define TAIL_SHAPES(VEC, CASE)                                                                                                                     \
    {                                                                                                                                              \
        const int nch = a.C / VEC;                                                                                                                 \
        if (nch <= 64) CASE(64, 1, VEC)                                                                                                            \
        else if (nch <= 128) CASE(64, 2, VEC)                                                                                                      \
        else if (nch <= 256) CASE(64, 4, VEC)                                                                                                      \
        else if (nch <= 512) CASE(256, 2, VEC)                                                                                                     \
        else if (nch <= 1024) CASE(256, 4, VEC)                                                                                                    \
        else if (nch <= 4096) CASE(1024, 4, VEC)                                                                                                   \
        else CASE(1024, 8, VEC)                                                                                                                    \
    }

template <typename T> void tail_fwd_launch(const TailArgs& a, bool vec, hipStream_t st) {
    const long rows = a.inner * a.outer;
#define FWD_CASE(TPR, NI, VEC)                                                                                             \
    {                                                                                                                      \
        constexpr int rpb = block_of<TPR>() / TPR;                                                                         \
        const long want = (rows + rpb - 1) / rpb, cap = 8L * hw_cu_count();                                                \
        hipLaunchKernelGGL((tail_fwd_kernel<T, TPR, NI, VEC>), dim3((unsigned)(want < cap ? want : cap)), dim3(block_of<TPR>()), 0, st, a); \
    }
    if (vec) TAIL_SHAPES(4, FWD_CASE)
    else TAIL_SHAPES(1, FWD_CASE)
#undef FWD_CASE
}
template <typename T> void tail_bwd_launch(const TailArgs& a, bool vec, int slices, hipStream_t st) {
    const bool full = a.res || a.gate || a.s || a.w2 || !a.w;
#define BWD_CASE(TPR, NI, VEC)                                                                                                                  \
    {                                                                                                                                           \
        if (full) hipLaunchKernelGGL((tail_bwd_kernel<T, TPR, NI, VEC, true>), dim3(slices, a.outer), dim3(block_of<TPR>()), 0, st, a);         \
        else hipLaunchKernelGGL((tail_bwd_kernel<T, TPR, NI, VEC, false>), dim3(slices, a.outer), dim3(block_of<TPR>()), 0, st, a);             \
    }
    if (vec) TAIL_SHAPES(4, BWD_CASE)
    else TAIL_SHAPES(1, BWD_CASE)
#undef BWD_CASE
}

bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

int tail_check(const char* what, const TailArgs& a) {
    HA2G_REQUIRE(a.C >= 1 && a.C <= 16384 && a.G >= 1 && a.C % a.G == 0, "%s: C=%d in %d groups (C <= 16384)", what, a.C, a.G);
    HA2G_REQUIRE(a.outer >= 0 && a.inner >= 0 && a.outer <= 65535, "%s: %d sequences of %ld rows (at most 65535)", what, a.outer, a.inner);
    HA2G_REQUIRE(a.act == 0 || a.act == 3 || a.act == 4, "%s: activation %d", what, a.act);
    return 0;
}

}  // namespace

extern "C" {

// slices of a sequence's rows in the backward pass: ~2 blocks per compute unit over all sequences
int ha2g_block_tail_slices(int outer, long inner, int C) {
    if (outer < 1 || inner < 1) return 1;
    const long rpb = C <= 1024 ? 4 : 1;
    long s = (2L * hw_cu_count() + outer - 1) / outer;
    const long most = (inner + rpb - 1) / rpb;
    return (int)(s < 1 ? 1 : (s < most ? s : most));
}

int ha2g_block_tail_fwd(const void* y, const void* res, const void* gate, const float* w, const float* b, const float* s, const float* w2, const float* b2,
                        void* h, void* z, float* mu, float* rs, float* mu2, float* rs2, int outer, long inner, int gate_shared, int C, int G, int layer,
                        int act, float alpha, float eps, int b16_io, void* stream) {
    TailArgs a = {};
    a.y = y; a.res = res; a.gate = gate; a.w = w; a.b = b; a.s = s; a.w2 = w2; a.b2 = b2; a.h = h; a.z = z;
    a.mu = mu; a.rs = rs; a.mu2 = mu2; a.rs2 = rs2;
    a.outer = outer; a.inner = inner; a.gate_shared = gate_shared; a.C = C; a.G = G; a.layer = layer; a.act = act; a.alpha = alpha; a.eps = eps;
    if (const int rc = tail_check("block_tail_fwd", a)) return rc;
    if (outer == 0 || inner == 0) return 0;
    HA2G_REQUIRE(y && h && (!w2 || z) && (!layer || !rs || mu) && (!layer || !rs2 || mu2), "block_tail_fwd: null operand");
    const size_t e = b16_io ? 8 : 16;
    const bool vec = (C / G) % 4 == 0 && aligned(y, e) && aligned(res, e) && aligned(gate, e) && aligned(h, e) && aligned(z, e) && aligned(w, 16) &&
                     aligned(b, 16) && aligned(s, 16) && aligned(w2, 16) && aligned(b2, 16);
    HA2G_REQUIRE(vec || C <= 8192, "block_tail_fwd: C=%d > 8192 needs groups of a multiple of 4 and 16-byte aligned operands", C);
    if (b16_io) tail_fwd_launch<b16>(a, vec, (hipStream_t)stream);
    else tail_fwd_launch<float>(a, vec, (hipStream_t)stream);
    HA2G_CHECK_LAUNCH("block_tail_fwd");
    return 0;
}

int ha2g_block_tail_bwd(const void* y, const void* res, const void* gate, const float* w, const float* b, const float* s, const float* w2, const float* b2,
                        const float* mu, const float* rs, const float* mu2, const float* rs2, const void* dh, const void* dz, void* dy, void* dres,
                        void* dgate, float* part, float* gpart, float* dparams, int slices, int outer, long inner, int gate_shared, int C, int G,
                        int layer, int act, float alpha, float eps, int b16_io, void* stream) {
    TailArgs a = {};
    a.y = y; a.res = res; a.gate = gate; a.w = w; a.b = b; a.s = s; a.w2 = w2; a.b2 = b2;
    a.mu = const_cast<float*>(mu); a.rs = const_cast<float*>(rs); a.mu2 = const_cast<float*>(mu2); a.rs2 = const_cast<float*>(rs2);
    a.dh = dh; a.dz = dz; a.dy = dy; a.dres = dres; a.dgate = dgate; a.part = part; a.gpart = gpart;
    a.outer = outer; a.inner = inner; a.gate_shared = gate_shared; a.C = C; a.G = G; a.layer = layer; a.act = act; a.alpha = alpha; a.eps = eps;
    if (const int rc = tail_check("block_tail_bwd", a)) return rc;
    HA2G_REQUIRE(slices >= 1 && slices <= 65535 * 8, "block_tail_bwd: %d slices", slices);
    if (outer == 0 || inner == 0) return 0;
    const int nvec = (w ? 2 : 0) + (s ? 1 : 0) + (w2 ? 2 : 0);
    HA2G_REQUIRE(y && (!w || rs) && (!w2 || rs2) && (!layer || !w || mu) && (!layer || !w2 || mu2) && (nvec == 0 || (part && dparams)) &&
                 (!(gate && gate_shared) || (gpart && dgate)), "block_tail_bwd: null operand");
    const size_t e = b16_io ? 8 : 16;
    const bool vec = (C / G) % 4 == 0 && aligned(y, e) && aligned(res, e) && aligned(gate, e) && aligned(dh, e) && aligned(dz, e) && aligned(dy, e) &&
                     aligned(dres, e) && aligned(dgate, e) && aligned(w, 16) && aligned(b, 16) && aligned(s, 16) && aligned(w2, 16) && aligned(b2, 16) &&
                     aligned(part, 16) && aligned(gpart, 16);
    HA2G_REQUIRE(vec || C <= 8192, "block_tail_bwd: C=%d > 8192 needs groups of a multiple of 4 and 16-byte aligned operands", C);
    const hipStream_t st = (hipStream_t)stream;
    if (b16_io) tail_bwd_launch<b16>(a, vec, slices, st);
    else tail_bwd_launch<float>(a, vec, slices, st);
    HA2G_CHECK_LAUNCH("block_tail_bwd");
    if (nvec) {
        hipLaunchKernelGGL(slab_sum_kernel<float>, dim3((nvec * C + 63) / 64), dim3(1024), 0, st, part, dparams, slices * outer, nvec * C);
        HA2G_CHECK_LAUNCH("block_tail_bwd: parameter sums");
    }
    if (gate && gate_shared) {
        const dim3 grid((C + 63) / 64, outer);
        if (b16_io) hipLaunchKernelGGL(slab_sum_kernel<b16>, grid, dim3(1024), 0, st, gpart, (b16*)dgate, slices, C);
        else hipLaunchKernelGGL(slab_sum_kernel<float>, grid, dim3(1024), 0, st, gpart, (float*)dgate, slices, C);
        HA2G_CHECK_LAUNCH("block_tail_bwd: gate sums");
    }
    return 0;
}

}  // extern "C"
