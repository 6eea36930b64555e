// Row norms and the tail of a block, forward and backward.  A row of C values is normalised in G groups of C / G (all of it, or per head):
//     RMS:   x^ = x / sqrt(mean(x^2) + eps)          layer:  x^ = (x - mean(x)) / sqrt(mean((x - mean)^2) + eps)
//     n = x^ w + b;   u = n act(gate);   h = alpha res + s u;   z = norm(h) w2 + b2   (over the whole row)
// Everything behind `n` is optional.  Statistics, products and sums are fp32 (the columns' sums over the rows end in double); h, z and the
// gradients are rounded once where they are stored, and z is the norm of h BEFORE that rounding, in the backward pass as in the forward one
// (h is formed again from y, res and gate there: the same bytes as reading h, and the parameters' gradients stay fp32-exact).
// Bound by HBM: a row lives in the registers of TPR threads (NI chunks of VEC values each) between its one read and its one write.
// Measured (bf16): 8 192 rows of 4 096 in 32 groups forward 31 us (4.3 TB/s; a large copy 4.9), backward 49 us (4.1 TB/s); 16 384 rows of 2 048 with
// everything behind the norm forward 66 us (336 MB, 5.1 TB/s), backward 128 us (537 MB, 4.2 TB/s: five of eight operands read, three written, and
// two rounds of row sums per row).
// Groups of a multiple of 16 bytes at aligned addresses are the straight case; otherwise (RAG: heads of 71, rows of 5 270) a chunk is four values at any
// address -- memory takes unaligned 16 bytes -- that may belong to two groups, and the row's last one may be short.
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
    float *rowsum;                   // [rows][2] the second norm's sums over a row (wide rows)
    float *gpart;                    // [outer][slices][C] sums of the gate's gradient over the slice's rows (gate shared by a sequence's rows)
    long inner;                      // rows of a sequence (= all rows where the gate is per row)
    int outer, C, G, layer, act, gate_shared;
    float alpha, eps;
};

// VEC values as they lie in memory, 16 bytes at most; ALIGN: at any multiple of a value's size
typedef unsigned u32x4u_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2u_t __attribute__((ext_vector_type(2)));
typedef u32x4u_t u32x4_a2 __attribute__((aligned(2)));
typedef u32x2u_t u32x2_a2 __attribute__((aligned(2)));
template <typename T, int VEC> struct Raw { unsigned u[(VEC * sizeof(T) + 3) / 4]; };
template <typename T, int VEC> __device__ __forceinline__ Raw<T, VEC> load_raw(const T* p, long at) {
    Raw<T, VEC> r;
    if constexpr (VEC * sizeof(T) == 16) { const u32x4_a2 v = *reinterpret_cast<const u32x4_a2*>(p + at); r.u[0] = v[0]; r.u[1] = v[1]; r.u[2] = v[2]; r.u[3] = v[3]; }
    else if constexpr (VEC * sizeof(T) == 8) { const u32x2_a2 v = *reinterpret_cast<const u32x2_a2*>(p + at); r.u[0] = v[0]; r.u[1] = v[1]; }
    else if constexpr (sizeof(T) == 4) r.u[0] = __float_as_uint(p[at]);
    else r.u[0] = p[at];
    return r;
}
// of which the first n exist (1 <= n <= VEC), zeros behind
template <typename T, int VEC> __device__ __forceinline__ Raw<T, VEC> load_raw(const T* p, long at, int n) {
    if (VEC == 1 || n == VEC) return load_raw<T, VEC>(p, at);
    Raw<T, VEC> r;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        if constexpr (sizeof(T) == 4) r.u[j] = j < n ? __float_as_uint(p[at + j]) : 0u;
        else {
            if (j % 2 == 0) r.u[j / 2] = 0u;
            if (j < n) r.u[j / 2] |= (unsigned)p[at + j] << (16 * (j & 1));
        }
    }
    return r;
}
template <int VEC> __device__ __forceinline__ void unpack(const Raw<float, VEC>& r, float* x) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = __uint_as_float(r.u[j]);
}
template <int VEC> __device__ __forceinline__ void unpack(const Raw<b16, VEC>& r, float* x) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = __uint_as_float((j & 1) ? r.u[j >> 1] & 0xffff0000u : r.u[j >> 1] << 16);
}
template <int VEC> __device__ __forceinline__ void store_row(float* p, long at, const float* x, int n = VEC) {
    if constexpr (VEC == 1) p[at] = x[0];
    else if (n == VEC) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
            const u32x4u_t v = {__float_as_uint(x[j]), __float_as_uint(x[j + 1]), __float_as_uint(x[j + 2]), __float_as_uint(x[j + 3])};
            *reinterpret_cast<u32x4_a2*>(p + at + j) = v;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < n) p[at + j] = x[j];
    }
}
template <int VEC> __device__ __forceinline__ void store_row(b16* p, long at, const float* x, int n = VEC) {
    unsigned h[(VEC + 1) / 2], l;
#pragma unroll
    for (int j = 0; j < VEC; j += 2) split2_bf16(x[j], VEC > 1 ? x[j + (VEC > 1)] : 0.f, h[j >> 1], l);
    if constexpr (VEC == 1) p[at] = (b16)(h[0] & 0xffff);
    else if (n == VEC) {
        if constexpr (VEC == 8) { const u32x4u_t v = {h[0], h[1], h[2], h[3]}; *reinterpret_cast<u32x4_a2*>(p + at) = v; }
        else { const u32x2u_t v = {h[0], h[1]}; *reinterpret_cast<u32x2_a2*>(p + at) = v; }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < n) p[at + j] = (b16)(h[j >> 1] >> (16 * (j & 1)));
    }
}
template <int VEC> __device__ __forceinline__ void load_vec(const float* p, long at, float* x, int n) {
    if constexpr (VEC == 8) { unpack<4>(load_raw<float, 4>(p, at), x); unpack<4>(load_raw<float, 4>(p, at + 4), x + 4); }
    else unpack<VEC>(load_raw<float, VEC>(p, at, n), x);
}
template <int VEC> __device__ __forceinline__ void fill(float* x, float v) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = v;
}

// Where a thread's chunks lie: values of chunk i that exist (n), its group, and how many of its values belong to that group (k; the rest to the next)
template <int TPR, int NI, int VEC, bool RAG> struct Place {
    int g[NI], k_[NI], n_[NI];
    __device__ __forceinline__ void init(const TailArgs& a, int lane) {
        const int D = a.C / a.G;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int at = (lane + i * TPR) * VEC;
            g[i] = at / D;
            if constexpr (RAG) {
                n_[i] = max(0, min(VEC, a.C - at));
                k_[i] = min(VEC, (g[i] + 1) * D - at);
            }
        }
    }
    __device__ __forceinline__ int n(int i) const { if constexpr (RAG) return n_[i]; else return VEC; }
    __device__ __forceinline__ int k(int i) const { if constexpr (RAG) return k_[i]; else return VEC; }
};

// 1 / (1 + e^-g) to 2^-22 of its value.  The hardware's 2^t of t = -g log2(e) rounded to fp32 is off by |g| 2^-24 of its value; what the rounding left out,
// r = -g - t ln 2 (ln 2 in two parts), enters as e^r = 1 + r.  t is held at 127, where r grows instead and the sum overflows as it should; an infinite g
// leaves r undefined and p infinite or 0: 0 for max(), which also takes a NaN for 0 (gate_act puts it back).
__device__ __forceinline__ float sigmoid_fp32(float g) {
    const float t = fminf(g * -1.44269504f, 127.f), p = __builtin_amdgcn_exp2f(t);
    const float r = __builtin_fmaf(t, 1.9046543e-9f, __builtin_fmaf(t, -0.693147182f, -g));
    return __builtin_amdgcn_rcpf(1.0f + fmaxf(__builtin_fmaf(p, r, p), 0.f));
}
// The gate's activation and its derivative.  Rows of fp32 take the sigmoid above (2^25 values: 2 048 per row, forward 137 us, 135 with the other, backward
// 250 and 249; at most, 1 500 per row, forward 154 and 144).  Rows of bf16 take the hardware's exponential and reciprocal: off by (|g| + 4) 2^-24 of
// the value, at most 2^-17 where the result is not 0 or 1, and every result of it is rounded to 2^-9 or summed in fp32 with errors of that size (the
// other one costs 3 to 10 %, and 60 % where it exceeds the registers: 1 500 and 2 002 values per row, backward 233 -> 366 and 261 -> 424 us).
template <typename T> __device__ __forceinline__ void gate_act(float g, int act, float& a, float& d) {
    if (act == 0) { a = g; d = 1.f; return; }
    float s;
    if constexpr (sizeof(T) == 4) {
        s = sigmoid_fp32(g);
        if (act == 3) s = g == g ? s : g;
    } else s = sigmoidf_(g);
    a = act == 3 ? s : g * s;
    d = act == 3 ? s * (1.f - s) : s * (1.f + g * (1.f - s));
}

// Sums over the row's TPR threads of a value per chunk (RAG: of its two parts): r = the sum over the group the chunk (its part) belongs to.  The whole
// row: a butterfly, and beyond a wave one meeting in LDS (two places in turn).  Groups of 2^n <= 64 chunks: a butterfly over their lanes.  Others
// (heads of 60): every chunk's value goes to LDS, a team of lanes adds up a group, its sum is read back.  A row of one wave needs no barrier.
// Every thread of the block calls it the same number of times.
template <int TPR, int NI, int VEC, bool RAG> struct RowSum {
    static constexpr int PARTS = RAG ? 2 : 1, PLACES = TPR * NI * PARTS + (RAG ? TPR * NI * VEC / 3 + 1 : 0);      // groups of 3 or more values
    float *lds, *meet;           // this row's PLACES floats; two times TPR / 64
    int lane, G, D, nch, phase;  // thread of the row, groups, values per group, chunks
    __device__ __forceinline__ static void sync() {
        if constexpr (TPR > 64) __syncthreads();
        else { __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront"); __builtin_amdgcn_wave_barrier(); __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront"); }
    }
    __device__ __forceinline__ float all(float s) {
        s = wave_sum(s);
        if constexpr (TPR > 64) {
            float* m = meet + phase * (TPR / 64);
            phase ^= 1;
            if ((lane & 63) == 0) m[lane >> 6] = s;
            __syncthreads();
            s = 0.f;
#pragma unroll
            for (int i = 0; i < TPR / 64; ++i) s += m[i];
        }
        return s;
    }
    __device__ __forceinline__ void groups(const Place<TPR, NI, VEC, RAG>& pl, const float (&p)[NI][PARTS], float (&r)[NI][PARTS]) {
        if (G == 1) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NI; ++i) s += p[i][0];
            s = all(s);
#pragma unroll
            for (int i = 0; i < NI; ++i) r[i][0] = r[i][PARTS - 1] = s;
            return;
        }
        const int cpg = D / VEC;
        if constexpr (!RAG)
            if (cpg <= 64 && (cpg & (cpg - 1)) == 0) {
#pragma unroll
                for (int i = 0; i < NI; ++i) r[i][0] = p[i][0];
                for (int o = cpg >> 1; o > 0; o >>= 1)
#pragma unroll
                    for (int i = 0; i < NI; ++i) r[i][0] += __shfl_xor(r[i][0], o, 64);
                return;
            }
        sync();
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            if (c < nch)
#pragma unroll
                for (int q = 0; q < PARTS; ++q) lds[c * PARTS + q] = p[i][q];
        }
        sync();
        const int team = G * 32 <= TPR ? 64 : 16;
        float* const sums = RAG ? lds + TPR * NI * PARTS : lds;
        for (int g = lane / team; g < G; g += TPR / team) {
            const int c0 = g * D / VEC, c1 = ((g + 1) * D + VEC - 1) / VEC;
            float s = 0.f;
            for (int c = c0 + lane % team; c < c1; c += team) s += lds[c * PARTS + (RAG && c * VEC < g * D ? 1 : 0)];
            for (int o = team >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
            if (lane % team == 0) sums[RAG ? g : c0] = s;
        }
        sync();
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            if constexpr (RAG) {
                r[i][0] = c < nch ? sums[pl.g[i]] : 0.f;
                r[i][1] = c < nch && pl.k(i) < pl.n(i) ? sums[pl.g[i] + 1] : 0.f;
            } else r[i][0] = c < nch ? sums[pl.g[i] * cpg] : 0.f;
        }
    }
};
// a chunk's value j: which of its parts
template <bool RAG> __device__ __forceinline__ int part_of(int j, int k) { return RAG && j >= k ? 1 : 0; }
template <bool RAG, int PARTS> __device__ __forceinline__ float pick(const float (&r)[PARTS], int j, int k) {
    if constexpr (RAG) return j >= k ? r[1] : r[0];
    else return r[0];
}
template <bool RAG, int PARTS> __device__ __forceinline__ void add_to(float (&p)[PARTS], int j, int k, bool whole, float v) {
    if constexpr (RAG) { if (whole || j < k) p[0] += v; else p[1] += v; }
    else p[0] += v;
}

// x -> x^ in place; m / r: mean and 1 / std per chunk and part.  Values that do not exist are zeros and stay zeros: their r is 0, not the 1 / sqrt(eps)
// of an empty sum, which is infinite for eps = 0.
template <int TPR, int NI, int VEC, bool RAG>
__device__ __forceinline__ void normalise(RowSum<TPR, NI, VEC, RAG>& rsum, const Place<TPR, NI, VEC, RAG>& pl, float (&x)[NI][VEC],
                                          float (&m)[NI][RowSum<TPR, NI, VEC, RAG>::PARTS], float (&r)[NI][RowSum<TPR, NI, VEC, RAG>::PARTS], bool layer,
                                          float inv, float eps) {
    constexpr int PARTS = RowSum<TPR, NI, VEC, RAG>::PARTS;
    const bool whole = rsum.G == 1;
    float p[NI][PARTS];
#pragma unroll
    for (int i = 0; i < NI; ++i) fill<PARTS>(m[i], 0.f);
    if (layer) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            fill<PARTS>(p[i], 0.f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) add_to<RAG>(p[i], j, pl.k(i), whole, x[i][j]);
        }
        rsum.groups(pl, p, m);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
#pragma unroll
            for (int q = 0; q < PARTS; ++q) m[i][q] *= inv;
            const bool in = rsum.lane + i * TPR < rsum.nch;
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[i][j] = in && j < pl.n(i) ? x[i][j] - pick<RAG>(m[i], j, pl.k(i)) : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        fill<PARTS>(p[i], 0.f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) add_to<RAG>(p[i], j, pl.k(i), whole, x[i][j] * x[i][j]);
    }
    rsum.groups(pl, p, r);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const bool in = rsum.lane + i * TPR < rsum.nch;
#pragma unroll
        for (int q = 0; q < PARTS; ++q) r[i][q] = in && (q == 0 || pl.k(i) < pl.n(i)) ? 1.0f / sqrtf(r[i][q] * inv + eps) : 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[i][j] *= pick<RAG>(r[i], j, pl.k(i));
    }
}

template <int TPR> constexpr int block_of() { return TPR > 256 ? TPR : 256; }

// The parameters' columns of a thread: kept in registers over the rows where a thread has one chunk, read from the caches per row otherwise.
template <int NI, int VEC> struct Columns {
    static constexpr bool KEEP = NI == 1;
    float w[VEC], b[VEC], s[VEC], w2[VEC], b2[VEC];
    __device__ __forceinline__ void load(const TailArgs& a, long at, bool in, int n) {
        fill<VEC>(w, 1.f); fill<VEC>(b, 0.f); fill<VEC>(s, 1.f); fill<VEC>(w2, 0.f); fill<VEC>(b2, 0.f);
        if (!in) return;
        if (a.w) load_vec<VEC>(a.w, at, w, n);
        if (a.b) load_vec<VEC>(a.b, at, b, n);
        if (a.s) load_vec<VEC>(a.s, at, s, n);
        if (a.w2) load_vec<VEC>(a.w2, at, w2, n);
        if (a.b2) load_vec<VEC>(a.b2, at, b2, n);
    }
};

template <typename T, int TPR, int NI, int VEC, bool RAG>
__global__ __launch_bounds__(block_of<TPR>()) void tail_fwd_kernel(const TailArgs a) {
    typedef RowSum<TPR, NI, VEC, RAG> Sum;
    constexpr int RPB = block_of<TPR>() / TPR;
    __shared__ float lds[RPB * Sum::PLACES], meet[RPB][2][2 * (TPR / 64)];
    const int sub = threadIdx.x / TPR, lane = threadIdx.x % TPR, nch = (a.C + VEC - 1) / VEC;
    const long rows = a.inner * a.outer;
    float* const mine = lds + sub * Sum::PLACES;
    Sum gsum{mine, meet[sub][0], lane, a.G, a.C / a.G, nch, 0}, rsum{mine, meet[sub][1], lane, 1, a.C, nch, 0};
    Place<TPR, NI, VEC, RAG> pl;
    pl.init(a, lane);
    Columns<NI, VEC> col;
    if constexpr (Columns<NI, VEC>::KEEP) col.load(a, (long)lane * VEC, lane < nch, pl.n(0));
    for (long r0 = (long)blockIdx.x * RPB; r0 < rows; r0 += (long)gridDim.x * RPB) {
        const long row = r0 + sub;
        const bool in = row < rows;
        const long at = row * a.C, gat = a.gate_shared ? row / a.inner * a.C : at;
        Raw<T, VEC> ry[NI], rg[NI], rr[NI];
        float x[NI][VEC], m[NI][Sum::PARTS], r[NI][Sum::PARTS];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            if (in && c < nch) {
                ry[i] = load_raw<T, VEC>((const T*)a.y, at + (long)c * VEC, pl.n(i));
                if (a.gate) rg[i] = load_raw<T, VEC>((const T*)a.gate, gat + (long)c * VEC, pl.n(i));
                if (a.res) rr[i] = load_raw<T, VEC>((const T*)a.res, at + (long)c * VEC, pl.n(i));
            }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            fill<VEC>(x[i], 0.f);
            if (in && c < nch) unpack<VEC>(ry[i], x[i]);
        }
        if (a.w) {
            normalise(gsum, pl, x, m, r, a.layer, (float)a.G / a.C, a.eps);
            if (a.rs && in) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int c = lane + i * TPR;
                    const long at = row * a.G + pl.g[i];              // a group's statistics are kept by the chunk it begins in
                    if (c < nch && c * VEC == pl.g[i] * gsum.D) {
                        a.rs[at] = r[i][0];
                        if (a.layer) a.mu[at] = m[i][0];
                    }
                    if (RAG && c < nch && pl.k(i) < pl.n(i)) {
                        a.rs[at + 1] = r[i][Sum::PARTS - 1];
                        if (a.layer) a.mu[at + 1] = m[i][Sum::PARTS - 1];
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            if (!(in && c < nch)) continue;
            if constexpr (!Columns<NI, VEC>::KEEP) col.load(a, (long)c * VEC, true, pl.n(i));
            float t[VEC];
            if (a.w) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][j] = x[i][j] * col.w[j] + col.b[j];
            }
            if (a.gate) {
                unpack<VEC>(rg[i], t);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { float ga, gd; gate_act<T>(t[j], a.act, ga, gd); x[i][j] *= ga; }
            }
            if (a.s) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][j] *= col.s[j];
            }
            if (a.res) {
                unpack<VEC>(rr[i], t);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][j] = a.alpha * t[j] + x[i][j];
            }
            if constexpr (RAG)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (j >= pl.n(i)) x[i][j] = 0.f;
            store_row<VEC>((T*)a.h, at + (long)c * VEC, x[i], pl.n(i));
        }
        if (a.w2) {
            normalise(rsum, pl, x, m, r, a.layer, 1.0f / a.C, a.eps);
            if (a.rs2 && in && lane == 0) {
                a.rs2[row] = r[0][0];
                if (a.layer) a.mu2[row] = m[0][0];
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = lane + i * TPR;
                if (!(in && c < nch)) continue;
                if constexpr (!Columns<NI, VEC>::KEEP) col.load(a, (long)c * VEC, true, pl.n(i));
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][j] = x[i][j] * col.w2[j] + col.b2[j];
                store_row<VEC>((T*)a.z, at + (long)c * VEC, x[i], pl.n(i));
            }
        }
    }
}

// One row's operands on their way: loaded a row ahead, so that a row's sums and barriers lie under the next row's loads
template <typename T, int TPR, int NI, int VEC, bool RAG, bool FULL> struct RowIn {
    static constexpr int PARTS = RAG ? 2 : 1;
    Raw<T, VEC> y[NI], dh[NI], dz[FULL ? NI : 1], gate[FULL ? NI : 1], res[FULL ? NI : 1];
    float mu[NI][PARTS], rs[NI][PARTS], mu2, rs2;
    __device__ __forceinline__ void load(const TailArgs& a, long row, long gat, bool in, int lane, int nch, const Place<TPR, NI, VEC, RAG>& pl) {
        mu2 = rs2 = 0.f;
        const long at = row * a.C;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            fill<PARTS>(mu[i], 0.f);
            fill<PARTS>(rs[i], 0.f);
            if (!(in && c < nch)) continue;
            y[i] = load_raw<T, VEC>((const T*)a.y, at + (long)c * VEC, pl.n(i));
            if (a.dh) dh[i] = load_raw<T, VEC>((const T*)a.dh, at + (long)c * VEC, pl.n(i));
            if (a.w) {
                const long g = row * a.G + pl.g[i];
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
                    if (q == 0 || pl.k(i) < pl.n(i)) {
                        rs[i][q] = a.rs[g + q];
                        if (a.layer) mu[i][q] = a.mu[g + q];
                    }
            }
            if constexpr (FULL) {
                if (a.dz) dz[i] = load_raw<T, VEC>((const T*)a.dz, at + (long)c * VEC, pl.n(i));
                if (a.gate) gate[i] = load_raw<T, VEC>((const T*)a.gate, gat + (long)c * VEC, pl.n(i));
                if (a.res && a.w2) res[i] = load_raw<T, VEC>((const T*)a.res, at + (long)c * VEC, pl.n(i));
            }
        }
        if constexpr (FULL) {
            if (a.w2 && in) {
                rs2 = a.rs2[row];
                if (a.layer) mu2 = a.mu2[row];
            }
        }
    }
};

// A block walks through the rows of its slice of a sequence and keeps the columns' sums in registers; its partial sums leave it once (128 sequences
// of 34 rows of 300: 18 us, the latency of five rounds of two rows, each with its sums across two waves).
// FULL: with gate, scale, residual or second norm; otherwise the norm alone (w, b).
template <typename T, int TPR, int NI, int VEC, bool RAG, bool FULL>
__global__ __launch_bounds__(block_of<TPR>()) void tail_bwd_kernel(const TailArgs a) {
    constexpr int RPB = block_of<TPR>() / TPR, NV = FULL ? 6 : 2;      // w, b, s, w2, b2, gate
    typedef RowSum<TPR, NI, VEC, RAG> Sum;
    constexpr int COLS = RPB > 1 ? RPB * TPR * NI * VEC : 1;
    __shared__ __attribute__((aligned(16))) float lds[RPB * Sum::PLACES > COLS ? RPB * Sum::PLACES : COLS];
    __shared__ float meet[RPB][2][2 * (TPR / 64)];
    const int sub = threadIdx.x / TPR, lane = threadIdx.x % TPR, nch = (a.C + VEC - 1) / VEC;
    float* const mine = lds + sub * Sum::PLACES;
    Sum gsum{mine, meet[sub][0], lane, a.G, a.C / a.G, nch, 0}, rsum{mine, meet[sub][1], lane, 1, a.C, nch, 0};
    Place<TPR, NI, VEC, RAG> pl;
    pl.init(a, lane);
    const bool whole = a.G == 1;
    const long per = (a.inner + gridDim.x - 1) / gridDim.x, beg = blockIdx.x * per, end = min(a.inner, beg + per);
    const float inv = (float)a.G / a.C, inv2 = 1.0f / a.C;
    const long row0 = (long)blockIdx.y * a.inner, gat0 = (long)blockIdx.y * a.C;
    float acc[NV][NI][VEC];
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < NI; ++i) fill<VEC>(acc[n][i], 0.f);
    Columns<NI, VEC> col;
    if constexpr (Columns<NI, VEC>::KEEP) col.load(a, (long)lane * VEC, lane < nch, pl.n(0));
    RowIn<T, TPR, NI, VEC, RAG, FULL> cur, nxt;
    cur.load(a, row0 + beg + sub, a.gate_shared ? gat0 : (row0 + beg + sub) * a.C, beg + sub < end, lane, nch, pl);
    for (long q0 = beg; q0 < end; q0 += RPB) {
        const bool in = q0 + sub < end;
        const long row = row0 + q0 + sub, at = row * a.C;
        nxt.load(a, row + RPB, a.gate_shared ? gat0 : (row + RPB) * a.C, q0 + RPB + sub < end, lane, nch, pl);
        float xh[NI][VEC], n[NI][VEC], d[NI][VEC], ga[FULL ? NI : 1][VEC], gd[FULL ? NI : 1][VEC];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            fill<VEC>(xh[i], 0.f); fill<VEC>(n[i], 0.f); fill<VEC>(d[i], 0.f);
            if constexpr (FULL) { fill<VEC>(ga[i], 1.f); fill<VEC>(gd[i], 0.f); }
            if (!(in && c < nch)) continue;
            if constexpr (!Columns<NI, VEC>::KEEP) col.load(a, (long)c * VEC, true, pl.n(i));
            unpack<VEC>(cur.y[i], xh[i]);
            if (a.dh) unpack<VEC>(cur.dh[i], d[i]);
            if (a.w) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) xh[i][j] = (xh[i][j] - pick<RAG>(cur.mu[i], j, pl.k(i))) * pick<RAG>(cur.rs[i], j, pl.k(i));
            }
            if constexpr (FULL) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) n[i][j] = a.w ? xh[i][j] * col.w[j] + col.b[j] : xh[i][j];
                if (a.gate) {
                    float t[VEC];
                    unpack<VEC>(cur.gate[i], t);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) gate_act<T>(t[j], a.act, ga[i][j], gd[i][j]);
                }
            }
        }
        if constexpr (FULL) {
            if (a.w2) {
                float hh[NI][VEC], e[NI][VEC], s1 = 0.f, s2 = 0.f;
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int c = lane + i * TPR;
                    fill<VEC>(hh[i], 0.f); fill<VEC>(e[i], 0.f);
                    if (!(in && c < nch)) continue;
                    if constexpr (!Columns<NI, VEC>::KEEP) col.load(a, (long)c * VEC, true, pl.n(i));
                    float t[VEC];
                    fill<VEC>(t, 0.f);
                    if (a.res) unpack<VEC>(cur.res[i], t);
                    if (a.dz) unpack<VEC>(cur.dz[i], e[i]);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        float h = n[i][j] * ga[i][j];
                        if (a.s) h *= col.s[j];
                        if (a.res) h = a.alpha * t[j] + h;
                        hh[i][j] = j < pl.n(i) ? (h - cur.mu2) * cur.rs2 : 0.f;
                        acc[3][i][j] += e[i][j] * hh[i][j];
                        acc[4][i][j] += e[i][j];
                        e[i][j] *= col.w2[j];
                        s1 += e[i][j] * hh[i][j];
                        s2 += e[i][j];
                    }
                }
                s1 = rsum.all(s1) * inv2;
                s2 = a.layer ? rsum.all(s2) * inv2 : 0.f;
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) d[i][j] += cur.rs2 * (e[i][j] - hh[i][j] * s1 - s2);
            }
        }
        // d = the whole gradient of h (of n, where there is nothing behind it) -> d(x^)
        float p1[NI][Sum::PARTS], p2[NI][Sum::PARTS];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            fill<Sum::PARTS>(p1[i], 0.f);
            fill<Sum::PARTS>(p2[i], 0.f);
            if constexpr (RAG)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (j >= pl.n(i)) d[i][j] = 0.f;
            if (!(in && c < nch)) { fill<VEC>(d[i], 0.f); continue; }
            if constexpr (!Columns<NI, VEC>::KEEP) col.load(a, (long)c * VEC, true, pl.n(i));
            if constexpr (FULL) {
                float t[VEC];
                if (a.dres) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) t[j] = a.alpha * d[i][j];
                    store_row<VEC>((T*)a.dres, at + (long)c * VEC, t, pl.n(i));
                }
                if (a.s) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) { acc[2][i][j] += d[i][j] * (n[i][j] * ga[i][j]); d[i][j] *= col.s[j]; }
                }
                if (a.gate) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        t[j] = d[i][j] * n[i][j] * gd[i][j];
                        acc[5][i][j] += t[j];
                        d[i][j] *= ga[i][j];
                    }
                    if (a.dgate && !a.gate_shared) store_row<VEC>((T*)a.dgate, at + (long)c * VEC, t, pl.n(i));
                }
            }
            if (a.w) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    acc[0][i][j] += d[i][j] * xh[i][j];
                    acc[1][i][j] += d[i][j];
                    d[i][j] *= col.w[j];
                    add_to<RAG>(p1[i], j, pl.k(i), whole, d[i][j] * xh[i][j]);
                    add_to<RAG>(p2[i], j, pl.k(i), whole, d[i][j]);
                }
            }
        }
        if (a.w) {
            float c1[NI][Sum::PARTS], c2[NI][Sum::PARTS];
            gsum.groups(pl, p1, c1);
            if (a.layer) gsum.groups(pl, p2, c2);
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    d[i][j] = pick<RAG>(cur.rs[i], j, pl.k(i)) * (d[i][j] - xh[i][j] * (pick<RAG>(c1[i], j, pl.k(i)) * inv) - (a.layer ? pick<RAG>(c2[i], j, pl.k(i)) * inv : 0.f));
        }
        if (a.dy) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = lane + i * TPR;
                if (in && c < nch) store_row<VEC>((T*)a.dy, at + (long)c * VEC, d[i], pl.n(i));
            }
        }
        cur = nxt;
    }
    const bool have[6] = {a.w != nullptr, a.w != nullptr, a.s != nullptr, a.w2 != nullptr, a.w2 != nullptr, a.gate_shared && a.gpart};
    int nvec = 0, k = 0;
#pragma unroll
    for (int q = 0; q < 5; ++q) nvec += have[q];
    const long blk = (long)blockIdx.y * gridDim.x + blockIdx.x;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        if (!have[q]) continue;
        float* out = q == 5 ? a.gpart + blk * a.C : a.part + (blk * nvec + k) * a.C;
        ++k;
        if constexpr (RPB > 1) {                     // the sums of the block's RPB rows meet in LDS, in the order of the rows
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = lane + i * TPR;
                if (c < nch)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) lds[(sub * NI * TPR + c) * VEC + j] = acc[q][i][j];
            }
            __syncthreads();
            for (int c = threadIdx.x; c < a.C; c += RPB * TPR) {
                float s = 0.f;
#pragma unroll
                for (int z = 0; z < RPB; ++z) s += lds[z * NI * TPR * VEC + c];
                out[c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = lane + i * TPR;
                if (c < nch) store_row<VEC>(out, (long)c * VEC, acc[q][i], pl.n(i));
            }
        }
    }
}

// What a chunk of a row is computed from
template <typename T, int VEC, bool RAG, bool FULL> struct ChunkIn {
    static constexpr int PARTS = RAG ? 2 : 1, V2 = FULL ? VEC : 1;
    Raw<T, VEC> y, dh;
    Raw<T, V2> dz, gate, res;
    float mu[PARTS], rs[PARTS];
    // the chunk at column c, of which n values exist, k of them in group g; row and gat (the gate's row) are the same for a whole wave
    __device__ __forceinline__ void load(const TailArgs& a, long row, long gat, unsigned c, unsigned g, int n, int k, bool in) {
        fill<PARTS>(mu, 0.f);
        fill<PARTS>(rs, 0.f);
        if (!in) return;
        const long at = row * a.C;
        y = load_raw<T, VEC>((const T*)a.y + at, c, n);
        if (a.dh) dh = load_raw<T, VEC>((const T*)a.dh + at, c, n);
        if (a.w) {
            const float *rsp = a.rs + row * a.G, *mup = a.mu + row * a.G;
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
                if (q == 0 || k < n) {
                    rs[q] = rsp[g + q];
                    if (a.layer) mu[q] = mup[g + q];
                }
        }
        if constexpr (FULL) {
            if (a.dz) dz = load_raw<T, VEC>((const T*)a.dz + at, c, n);
            if (a.gate) gate = load_raw<T, VEC>((const T*)a.gate + gat, c, n);
            if (a.res && a.w2) res = load_raw<T, VEC>((const T*)a.res + at, c, n);
        }
    }
};

// One chunk on its way back.  open(): x^, n, the gate's activation and derivative, and with a second norm h^ and dz.  back(): d = the whole gradient
// of h -> that of x^, what it adds to the columns' sums (w, b, s, w2, b2, gate), and the gradients of
// residual and gate at their places (nullptr = not wanted).
template <typename T, int VEC, bool RAG, bool FULL> struct Chunk {
    static constexpr int V2 = FULL ? VEC : 1, PARTS = RAG ? 2 : 1;
    float xh[VEC], n[V2], ga[V2], gd[V2], hh[V2], e[V2];
    template <int NI> __device__ __forceinline__ void open(const TailArgs& a, const ChunkIn<T, VEC, RAG, FULL>& in, const Columns<NI, VEC>& col, int have,
                                                           int k, float mu2, float rs2, bool there) {      // zeros where there is nothing
        fill<VEC>(xh, 0.f);
        if constexpr (FULL) { fill<VEC>(n, 0.f); fill<VEC>(ga, 1.f); fill<VEC>(gd, 0.f); fill<VEC>(hh, 0.f); fill<VEC>(e, 0.f); }
        if (!there) return;
        unpack<VEC>(in.y, xh);
        if (a.w) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) xh[j] = (xh[j] - pick<RAG>(in.mu, j, k)) * pick<RAG>(in.rs, j, k);
        }
        if constexpr (FULL) {
            float t[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) n[j] = a.w ? xh[j] * col.w[j] + col.b[j] : xh[j];
            if (a.gate) {
                unpack<VEC>(in.gate, t);
#pragma unroll
                for (int j = 0; j < VEC; ++j) gate_act<T>(t[j], a.act, ga[j], gd[j]);
            }
            if (a.w2) {
                fill<VEC>(t, 0.f);
                if (a.res) unpack<VEC>(in.res, t);
                if (a.dz) unpack<VEC>(in.dz, e);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float h = n[j] * ga[j];
                    if (a.s) h *= col.s[j];
                    if (a.res) h = a.alpha * t[j] + h;
                    hh[j] = j < have ? (h - mu2) * rs2 : 0.f;
                }
            }
        }
    }
    // what the second norm's gradient needs of the whole row
    template <int NI> __device__ __forceinline__ void second(const Columns<NI, VEC>& col, float& s1, float& s2) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float t = e[j] * col.w2[j];
            s1 += t * hh[j];
            s2 += t;
        }
    }
    template <int NI, int NA> __device__ __forceinline__ void back(const TailArgs& a, const ChunkIn<T, VEC, RAG, FULL>& in, const Columns<NI, VEC>& col, int have,
                                                                   float rs2, float s1, float s2, float (&d)[VEC], float (&acc)[NA][VEC], T* dres,
                                                                   T* dgate) const {
        constexpr bool SUMS = NA > 1;
        fill<VEC>(d, 0.f);
        if (a.dh) unpack<VEC>(in.dh, d);
        if constexpr (FULL)
            if (a.w2) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if constexpr (SUMS) { acc[3][j] += e[j] * hh[j]; acc[4][j] += e[j]; }
                    d[j] += rs2 * (e[j] * col.w2[j] - hh[j] * s1 - s2);
                }
            }
        if constexpr (RAG)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (j >= have) d[j] = 0.f;
        if constexpr (FULL) {
            float t[VEC];
            if (dres) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) t[j] = a.alpha * d[j];
                store_row<VEC>(dres, 0, t, have);
            }
            if (a.s) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if constexpr (SUMS) acc[2][j] += d[j] * (n[j] * ga[j]);
                    d[j] *= col.s[j];
                }
            }
            if (a.gate) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    t[j] = d[j] * n[j] * gd[j];
                    if constexpr (SUMS) acc[5][j] += t[j];
                    d[j] *= ga[j];
                }
                if (dgate) store_row<VEC>(dgate, 0, t, have);
            }
        }
        if (a.w) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if constexpr (SUMS) { acc[0][j] += d[j] * xh[j]; acc[1][j] += d[j]; }
                d[j] *= col.w[j];
            }
        }
    }
};

// Rows of more than a chunk for each of 1 024 threads, whose 128 registers do not hold the columns' sums as well: two kernels.  This one takes the rows:
// the chunks are opened one by one, once for the sums of the second norm, from the caches again for the rest; only x^ and its gradient are kept.
// The row's two sums go to memory for the other.  Two chunks' operands are kept in registers, four are read again (16 384 values of bf16: 333 us, kept
// and spilled 423).  8 192 values, 2^25 in all: bf16 199 us (2.7 TB/s), fp32 310 (3.5); bound by its one block per compute unit, whose loads, two
// row sums and stores follow one another.
template <typename T, int NI, bool RAG, bool FULL>
__global__ __launch_bounds__(1024) void tail_wide_kernel(const TailArgs a) {
    constexpr int TPR = 1024, VEC = 4;
    constexpr bool KEEP = NI == 2;      // its operands stay in registers, loaded once
    constexpr int KEPT = KEEP ? NI : 1;
    typedef RowSum<TPR, NI, VEC, RAG> Sum;
    __shared__ float lds[Sum::PLACES], meet[2][2 * (TPR / 64)];
    const int lane = threadIdx.x, nch = (a.C + VEC - 1) / VEC;
    Sum gsum{lds, meet[0], lane, a.G, a.C / a.G, nch, 0}, rsum{lds, meet[1], lane, 1, a.C, nch, 0};
    Place<TPR, NI, VEC, RAG> pl;
    pl.init(a, lane);
    const bool whole = a.G == 1;
    const long per = (a.inner + gridDim.x - 1) / gridDim.x, beg = (long)blockIdx.y * a.inner + blockIdx.x * per, end = (long)blockIdx.y * a.inner + min(a.inner, (blockIdx.x + 1) * per);
    const float inv = (float)a.G / a.C, inv2 = 1.0f / a.C;
    for (long row = beg; row < end; ++row) {
        const long at = row * a.C;
        float mu2 = 0.f, rs2 = 0.f, s1 = 0.f, s2 = 0.f, none[1][VEC];
        Columns<NI, VEC> col;
        ChunkIn<T, VEC, RAG, FULL> in[KEPT];
        Chunk<T, VEC, RAG, FULL> ch;
        auto load = [&](int i) {
            const int c = lane + i * TPR;
            in[KEEP ? i : 0].load(a, row, a.gate_shared ? (long)blockIdx.y * a.C : at, c * VEC, pl.g[i], pl.n(i), pl.k(i), c < nch);
        };
        auto open = [&](int i) {
            const int c = lane + i * TPR;
            __builtin_amdgcn_sched_barrier(0);                  // one chunk after another: the registers hold one
            if (c < nch) col.load(a, (long)c * VEC, true, pl.n(i));
            if constexpr (!KEEP) load(i);
            ch.open(a, in[KEEP ? i : 0], col, pl.n(i), pl.k(i), mu2, rs2, c < nch);
        };
        if constexpr (KEEP)
#pragma unroll
            for (int i = 0; i < NI; ++i) load(i);
        if constexpr (FULL)
            if (a.w2) {
                rs2 = a.rs2[row];
                if (a.layer) mu2 = a.mu2[row];
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    open(i);
                    if (lane + i * TPR < nch) ch.second(col, s1, s2);
                }
                s1 = rsum.all(s1) * inv2;
                s2 = a.layer ? rsum.all(s2) * inv2 : 0.f;
                if (lane == 0) { a.rowsum[2 * row] = s1; a.rowsum[2 * row + 1] = s2; }
            }
        float d[NI][VEC], xh[NI][VEC], p1[NI][Sum::PARTS], p2[NI][Sum::PARTS];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = lane + i * TPR;
            fill<Sum::PARTS>(p1[i], 0.f);
            fill<Sum::PARTS>(p2[i], 0.f);
            fill<VEC>(d[i], 0.f);
            open(i);
#pragma unroll
            for (int j = 0; j < VEC; ++j) xh[i][j] = ch.xh[j];
            if (c >= nch) continue;
            ch.back(a, in[KEEP ? i : 0], col, pl.n(i), rs2, s1, s2, d[i], none, FULL && a.dres ? (T*)a.dres + at + c * VEC : nullptr,
                    FULL && a.dgate && !a.gate_shared ? (T*)a.dgate + at + c * VEC : nullptr);
            if (a.w) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    add_to<RAG>(p1[i], j, pl.k(i), whole, d[i][j] * xh[i][j]);
                    add_to<RAG>(p2[i], j, pl.k(i), whole, d[i][j]);
                }
            }
        }
        if (a.w) {
            float c1[NI][Sum::PARTS], c2[NI][Sum::PARTS];
            gsum.groups(pl, p1, c1);
            if (a.layer) gsum.groups(pl, p2, c2);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                float rs[Sum::PARTS];
#pragma unroll
                for (int q = 0; q < Sum::PARTS; ++q) rs[q] = lane + i * TPR < nch && (q == 0 || pl.k(i) < pl.n(i)) ? a.rs[row * a.G + pl.g[i] + q] : 0.f;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    d[i][j] = pick<RAG>(rs, j, pl.k(i)) * (d[i][j] - xh[i][j] * (pick<RAG>(c1[i], j, pl.k(i)) * inv) - (a.layer ? pick<RAG>(c2[i], j, pl.k(i)) * inv : 0.f));
            }
        }
        if (a.dy) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = lane + i * TPR;
                if (c < nch) store_row<VEC>((T*)a.dy, at + (long)c * VEC, d[i], pl.n(i));
            }
        }
    }
}

// The columns' sums of wide rows: a block has 256 columns (four per lane) of a slice of a sequence's rows, which its four waves take in turn; the row
// sums are there already, so that nothing is shared until the end.  Bound by memory, five operands a second time: 8 192 values, 2^25 in all: bf16
// 75 us (4.5 TB/s), fp32 140 (4.8).
template <typename T, bool RAG>
__global__ __launch_bounds__(256) void tail_columns_kernel(const TailArgs a) {
    __shared__ __attribute__((aligned(16))) float lds[4 * 256];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c0 = blockIdx.x * 256, c = c0 + 4 * lane, D = a.C / a.G, g = c / D;
    const int n = RAG ? max(0, min(4, a.C - c)) : 4, k = RAG ? min(4, (g + 1) * D - c) : 4;
    const bool there = c < a.C;
    const long per = (a.inner + gridDim.y - 1) / gridDim.y, beg = blockIdx.y * per, end = min(a.inner, beg + per), row0 = (long)blockIdx.z * a.inner;
    float acc[6][4];
#pragma unroll
    for (int q = 0; q < 6; ++q) fill<4>(acc[q], 0.f);
    Columns<1, 4> col;
    col.load(a, c, there, n);
    for (long q = beg + wave; q < end; q += 4) {
        const long row = row0 + q;
        ChunkIn<T, 4, RAG, true> in;
        in.load(a, row, a.gate_shared ? (long)blockIdx.z * a.C : row * a.C, c, g, n, k, there);
        float mu2 = 0.f, rs2 = 0.f, s1 = 0.f, s2 = 0.f;
        if (a.w2) {
            rs2 = a.rs2[row];
            if (a.layer) mu2 = a.mu2[row];
            s1 = a.rowsum[2 * row];
            s2 = a.rowsum[2 * row + 1];
        }
        Chunk<T, 4, RAG, true> ch;
        ch.open(a, in, col, n, k, mu2, rs2, there);
        if (!there) continue;
        float d[4];
        ch.back(a, in, col, n, rs2, s1, s2, d, acc, (T*)nullptr, (T*)nullptr);
    }
    const bool have[6] = {a.w != nullptr, a.w != nullptr, a.s != nullptr, a.w2 != nullptr, a.w2 != nullptr, a.gate_shared && a.gpart};
    const long blk = (long)blockIdx.z * gridDim.y + blockIdx.y;
    int nvec = 0, at = 0;
#pragma unroll
    for (int q = 0; q < 5; ++q) nvec += have[q];
#pragma unroll
    for (int q = 0; q < 6; ++q) {
        if (!have[q]) continue;
        float* out = (q == 5 ? a.gpart + blk * a.C : a.part + (blk * nvec + at) * a.C) + c0;
        ++at;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) lds[wave * 256 + 4 * lane + j] = acc[q][j];
        __syncthreads();
        if (c0 + (int)threadIdx.x < a.C) out[threadIdx.x] = lds[threadIdx.x] + lds[256 + threadIdx.x] + lds[512 + threadIdx.x] + lds[768 + threadIdx.x];
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

// The forward pass: threads per row and chunks per thread.  A wave alone up to 128 chunks, then one chunk per thread as far as 256 threads go, then two; the
// widest rows take what the registers of 1 024 threads hold.  Ragged chunks cost more registers: one per thread up to 512 threads (2^25 values,
// fp32, before its sigmoid, which adds up to 7 %: 300 per row 199 us, 242 with two per thread; 1 500 145 us, 195; but 2 700 224 us with one in 1 024
// threads, 219 with two in 512).  Groups of one or two values (VEC = 1) are taken one by one.
#define TAIL_SHAPES(VEC, RAG, CASE)                                                                                                                \
    {                                                                                                                                              \
        const int nch = (a.C + VEC - 1) / VEC;                                                                                                     \
        if (nch <= 64) CASE(64, 1, VEC, RAG)                                                                                                       \
        else if (nch <= 128) CASE((RAG ? 128 : 64), (RAG ? 1 : 2), VEC, RAG)                                                                       \
        else if (nch <= 256) CASE(256, 1, VEC, RAG)                                                                                                \
        else if (nch <= 512) CASE((RAG ? 512 : 256), (RAG ? 1 : 2), VEC, RAG)                                                                      \
        else if (nch <= 1024) CASE(512, 2, VEC, RAG)                                                                                               \
        else if (nch <= 2048) CASE(1024, 2, VEC, RAG)                                                                                              \
        else CASE(1024, (VEC == 8 ? 2 : 4), VEC, RAG)                                                                                              \
    }
#define TAIL_ONES(CASE)                                                                                                                            \
    {                                                                                                                                              \
        if (a.C <= 1024) CASE(256, 4, 1, false)                                                                                                    \
        else CASE(1024, 16, 1, false)                                                                                                              \
    }
#define TAIL_VECS(CASE)                                                                                                                            \
    if (vec == 1) TAIL_ONES(CASE)                                                                                                                  \
    else if (rag) TAIL_SHAPES(4, true, CASE)                                                                                                       \
    else if constexpr (sizeof(T) == 2) {                                                                                                           \
        if (vec == 8) TAIL_SHAPES(8, false, CASE)                                                                                                  \
        else TAIL_SHAPES(4, false, CASE)                                                                                                           \
    } else TAIL_SHAPES(4, false, CASE)

template <typename T> void tail_fwd_launch(const TailArgs& a, int vec, bool rag, hipStream_t st) {
    const long rows = a.inner * a.outer;
#define FWD_CASE(TPR, NI, VEC, RAG)                                                                                        \
    {                                                                                                                      \
        constexpr int rpb = block_of<TPR>() / TPR;                                                                         \
        const long want = (rows + rpb - 1) / rpb, cap = 8L * hw_cu_count();                                                \
        hipLaunchKernelGGL((tail_fwd_kernel<T, TPR, NI, VEC, RAG>), dim3((unsigned)(want < cap ? want : cap)), dim3(block_of<TPR>()), 0, st, a); \
    }
    TAIL_VECS(FWD_CASE)
#undef FWD_CASE
}
// The backward pass.  With anything behind the norm a value costs some 25 registers, so a thread has one chunk of the row while 256 threads hold it, 512
// with chunks of eight or ragged ones, and two chunks of four beyond.  Measured on 2^25 values, us, the other choice behind it: bf16 1 024 values
// per row 136 (two chunks of eight in a wave: 211), 4 096 171 (two in 256 threads: 235; one of four in 1 024: 273); fp32 2 048 256 (one in 512
// threads: 268), 4 096 268 (one in 1 024: 426); ragged fp32 1 500 368 (two in 256: 550), 2 700 404 (one in 1 024: 436).
// Rows beyond 4 096 values, and the norm alone beyond 2 048 chunks, go to tail_wide_kernel and tail_columns_kernel: bf16 8 192 values 273 us (two chunks
// of eight in 1 024 threads, spilling: 392), 16 384 333 (1 020); fp32 8 192 443 (840), 16 384 581 (1 307), the norm alone there 124 (208).
bool tail_full(const TailArgs& a) { return a.dres || a.gate || a.s || a.w2 || !a.w; }
bool tail_wide(int C, int vec, bool full) { return vec > 1 && C > (full ? 4096 : 2048 * vec); }

template <typename T, bool RAG, bool FULL> void tail_wide_launch(const TailArgs& a, int slices, hipStream_t st) {
    const long want = (2L * hw_cu_count() + a.outer - 1) / a.outer;
    const dim3 grid((unsigned)(want < a.inner ? want : a.inner), a.outer), block(1024);
    bool two = false;                                             // the norm alone comes here with more than 8 192 values only
    if constexpr (FULL)
        if ((two = a.C <= 8192)) hipLaunchKernelGGL((tail_wide_kernel<T, 2, RAG, FULL>), grid, block, 0, st, a);
    if (!two) hipLaunchKernelGGL((tail_wide_kernel<T, 4, RAG, FULL>), grid, block, 0, st, a);
    if (a.w || a.s || a.w2 || (a.gate && a.gate_shared))
        hipLaunchKernelGGL((tail_columns_kernel<T, RAG>), dim3((a.C + 255) / 256, slices, a.outer), dim3(256), 0, st, a);
}
template <typename T, int TPR, int NI, int VEC, bool RAG, bool FULL> void tail_one_launch(const TailArgs& a, int slices, hipStream_t st) {
    hipLaunchKernelGGL((tail_bwd_kernel<T, TPR, NI, VEC, RAG, FULL>), dim3(slices, a.outer), dim3(block_of<TPR>()), 0, st, a);
}
template <typename T, int VEC, bool RAG> void tail_full_launch(const TailArgs& a, int slices, hipStream_t st) {
    const int nch = (a.C + VEC - 1) / VEC;
    if (nch <= 64) tail_one_launch<T, 64, 1, VEC, RAG, true>(a, slices, st);
    else if (nch <= 128) tail_one_launch<T, 128, 1, VEC, RAG, true>(a, slices, st);
    else if (nch <= 256) tail_one_launch<T, 256, 1, VEC, RAG, true>(a, slices, st);
    else if constexpr (VEC == 8) tail_one_launch<T, 512, 1, VEC, RAG, true>(a, slices, st);
    else if (RAG && nch <= 512) tail_one_launch<T, 512, 1, VEC, RAG, true>(a, slices, st);
    else if (nch <= 512) tail_one_launch<T, 256, 2, VEC, RAG, true>(a, slices, st);
    else tail_one_launch<T, 512, 2, VEC, RAG, true>(a, slices, st);
}
template <typename T, int VEC, bool RAG> void tail_norm_launch(const TailArgs& a, int slices, hipStream_t st) {
    const int nch = (a.C + VEC - 1) / VEC;
    if (nch <= 64) tail_one_launch<T, 64, 1, VEC, RAG, false>(a, slices, st);
    else if (nch <= 128) tail_one_launch<T, 64, 2, VEC, RAG, false>(a, slices, st);
    else if (nch <= 256) tail_one_launch<T, 256, 1, VEC, RAG, false>(a, slices, st);
    else if (nch <= 512) tail_one_launch<T, 256, 2, VEC, RAG, false>(a, slices, st);
    else if (nch <= 1024) tail_one_launch<T, 512, 2, VEC, RAG, false>(a, slices, st);
    else tail_one_launch<T, 1024, 2, VEC, RAG, false>(a, slices, st);
}
template <typename T, bool FULL> void tail_ones_launch(const TailArgs& a, int slices, hipStream_t st) {
    if (a.C <= 1024) tail_one_launch<T, 256, 4, 1, false, FULL>(a, slices, st);
    else tail_one_launch<T, 1024, 16, 1, false, FULL>(a, slices, st);
}
template <typename T> void tail_bwd_launch(const TailArgs& a, int vec, bool rag, int slices, hipStream_t st) {
    const bool full = tail_full(a), wide = tail_wide(a.C, vec, full);
    if (vec == 1) { if (full) tail_ones_launch<T, true>(a, slices, st); else tail_ones_launch<T, false>(a, slices, st); }
    else if (wide && rag) { if (full) tail_wide_launch<T, true, true>(a, slices, st); else tail_wide_launch<T, true, false>(a, slices, st); }
    else if (wide) { if (full) tail_wide_launch<T, false, true>(a, slices, st); else tail_wide_launch<T, false, false>(a, slices, st); }
    else if (rag) { if (full) tail_full_launch<T, 4, true>(a, slices, st); else tail_norm_launch<T, 4, true>(a, slices, st); }
    else {
        if constexpr (sizeof(T) == 2)
            if (vec == 8) return full ? tail_full_launch<T, 8, false>(a, slices, st) : tail_norm_launch<T, 8, false>(a, slices, st);
        if (full) tail_full_launch<T, 4, false>(a, slices, st); else tail_norm_launch<T, 4, false>(a, slices, st);
    }
}

// values per access (16 bytes' worth, bf16 also 8; 1 for groups of one or two values), and whether chunks may straddle groups or end short
int tail_vec(int C, int G, int b16_io, bool* rag) {
    const int D = C / G;
    *rag = false;
    if (G > 1 && D < 3) return 1;
    if (b16_io && D % 8 == 0) return 8;
    *rag = D % 4 != 0;
    return 4;
}

int tail_check(const char* what, const TailArgs& a) {
    HA2G_REQUIRE(a.C >= 1 && a.C <= 16384 && a.G >= 1 && a.C % a.G == 0, "%s: C=%d in %d groups (C <= 16384)", what, a.C, a.G);
    HA2G_REQUIRE(a.outer >= 0 && a.inner >= 0 && a.outer <= 65535, "%s: %d sequences of %ld rows (at most 65535)", what, a.outer, a.inner);
    HA2G_REQUIRE(a.act == 0 || a.act == 3 || a.act == 4, "%s: activation %d", what, a.act);
    return 0;
}

}  // namespace

extern "C" {

// slices of a sequence's rows in the backward pass: two blocks per compute unit over all sequences (one of 512 threads; four with 8-byte loads: bf16,
// 1 000 values in two groups 145 us, 211), each at least one turn of its rows.  More of them only write more sums (fp32, 1 024 values: 232 us with two
// blocks, 273 with four).
int ha2g_block_tail_slices(int outer, long inner, int C, int G, int full, int b16_io) {
    if (outer < 1 || inner < 1 || C < 1 || G < 1) return 1;
    bool rag;
    const int vec = tail_vec(C, G, b16_io, &rag);
    long want = 2L * hw_cu_count(), rows = C <= 256 ? 4 : (C <= 512 ? 2 : 1);
    if (tail_wide(C, vec, full != 0)) { want = 4L * hw_cu_count() / ((C + 255) / 256); rows = 16; }
    else if (full && C > 2048) want = hw_cu_count();
    else if (full && b16_io && vec == 4) want *= 2;              // 8-byte loads: more waves to have as much in flight
    const long s = (want + outer - 1) / outer, most = (inner + rows - 1) / rows;
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
    bool rag;
    const int vec = tail_vec(C, G, b16_io, &rag);
    if (b16_io) tail_fwd_launch<b16>(a, vec, rag, (hipStream_t)stream);
    else tail_fwd_launch<float>(a, vec, rag, (hipStream_t)stream);
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
    HA2G_REQUIRE(slices >= 1 && slices <= 65535, "block_tail_bwd: %d slices", slices);
    if (outer == 0 || inner == 0) return 0;
    const int nvec = (w ? 2 : 0) + (s ? 1 : 0) + (w2 ? 2 : 0);
    a.rowsum = part + (long)slices * outer * nvec * C;
    HA2G_REQUIRE(y && (!w || rs) && (!w2 || rs2) && (!layer || !w || mu) && (!layer || !w2 || mu2) && (nvec == 0 || (part && dparams)) &&
                 (!(gate && gate_shared) || (gpart && dgate)), "block_tail_bwd: null operand");
    bool rag;
    const int vec = tail_vec(C, G, b16_io, &rag);
    const hipStream_t st = (hipStream_t)stream;
    if (b16_io) tail_bwd_launch<b16>(a, vec, rag, slices, st);
    else tail_bwd_launch<float>(a, vec, rag, slices, st);
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
