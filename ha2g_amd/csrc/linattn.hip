// Linear attention with one decay per head: a recurrence over time whose state is a Dk x Dv matrix per head,
//     S_t = e^g S_{t-1} + k_t v_t^T,    o_t = scale * q_t S_t,    g <= 0 per head.
// The backward pass is the same recurrence on other operands (do = the gradient of o, P = the gradient of the last state):
//     dq = the forward recurrence on (do, v, k);  dk = the recurrence from the end on (v, do, q);  dv = the one from the end on (k, q, do),
// where a step from the end adds, reads and then decays (R = P + scale q do^T, out, P = e^g R): the gradient of the last state reaches the last
// token undecayed, and what is left in front of the first token is the gradient of the first state.
#include "common.h"

#include <climits>

namespace {

struct Operand { const void* p; long b, t, h; int r; };      // element strides of batch row, token, head; head h reads head h / r

// one recurrence: reads q k v, adds k v^T, writes o
struct Job {
    Operand q, k, v;
    void* o;
    long ob, ot, oh;
    const float* s_in;           // states in front of the first token, one after another for (b, h), element (i, j) at i * si + j * sj; nullptr = zero
    float* s_out;                // those behind the last one, laid out alike, or nullptr
    float* seg;                  // [B * H][nseg - 1] states between the segments, element (i, j) at i * gi + j * gj
    int si, sj, gi, gj, Dk, Dv, rev, o16;
    float oscale, uscale;        // on what is read, on what is added
};
struct LinAttnArgs {
    Job job[3];
    const float* g;              // [H] log decay
    const int* lengths;          // [B] tokens of each sequence, or nullptr = T
    int B, T, H, nseg, seg_len;  // segments of seg_len tokens (a multiple of the chunk)
};

template <typename T> __device__ __forceinline__ void st1(T* p, long i, float v);
template <> __device__ __forceinline__ void st1<float>(float* p, long i, float v) { p[i] = v; }
template <> __device__ __forceinline__ void st1<b16>(b16* p, long i, float v) {
    unsigned h, l;
    split2_bf16(v, 0.f, h, l);
    p[i] = (b16)(h & 0xffff);
}

// ---- chunked form --------------------------------------------------------------------------------------------------------------------------
// C tokens at a time (fp32: 32, bf16: 64; half of that for Dk > 64), positions i, j inside the chunk, e = 1 forward and 0 from the end:
//     o_i = e^{g (i + e)} q_i S + sum_{j <= i} e^{g (i - j)} (q_i k_j) v_j,        S <- e^{g C} S + sum_j e^{g (C - e - j)} k_j v_j^T
// A workgroup owns a (batch row, head, segment of the time axis); its waves split the columns of v, each keeps its Dk x DVW slice of S in MFMA
// accumulators for the whole segment.  The accumulator layout (column = lane & 15, row = 4 (lane >> 4) + i) is that of an operand whose k runs along
// the rows, up to an order of k that both operands may share: S goes from accumulators straight into the next product and is never laid out again.
// The scores k q^T are the same for all columns of v: each wave computes its share of their 16 x 16 tiles and leaves them in LDS as the next
// product's operands, for all.  Rows of LDS are padded by 32 bytes: 16-byte reads of 16 rows and transpose reads of 4 x 16 blocks meet every bank
// once (row reads of 2 x 8 bytes had two thirds of the LDS time in conflicts).
//     o^T = S^T q^T + v^T (k q^T):  a lane ends with 4 consecutive columns of one token.
// Measured: 512 (row, head) pairs of 1 024 tokens, bf16: Dk = Dv = 64 62 us (q, k, v and o at 4.3 TB/s; a large copy 4.9), 128 131 us (4.1 TB/s);
// fp32: 125 us (4.3 TB/s) and 365 us (2.9).  Bound by memory at 64, at 128 by the issue of two waves per SIMD: per chunk and wave ~500 vector
// instructions (200 of them split S, 64 decay it) beside 91 matrix instructions, matrix units 30 % busy.
// fp32 operands run on the fp32 MFMA.  bf16 operands are exact as they are; what is computed is split into bf16 pieces: S and the scores, which
// only reach the bf16 result, into two (2^-17 of a term, 2^-8 of the result's own rounding; a third piece costs 10 to 22 %: 512 pairs, 128 x 128,
// forward 160 us, 131, backward 429, 347), the decayed v that is added to S into three (all 24 bits: S stays fp32-exact).
// The decay of S is S + S (e^{gC} - 1) where more than half is kept: a factor rounded to fp32 is off the same way in every chunk, 1e-4 of a state with a
// memory of 2^12 tokens.  Where less is kept it is S e^{gC}: the sum is exact to 2^-24 of the S before, not of what is left of it.
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t* lds4_t;

template <typename T> struct Mma;
template <> struct Mma<float> {
    typedef f32x4 Frag;
    static constexpr int C = 32, KB = 16, PADK = 16, NS = 1, NV = 1;      // longest chunk, k per fragment, LDS row padding, pieces of S / scores and of v
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
    __device__ __forceinline__ static Frag state_col(const float* p, int ld, int x, int u, int lane) { return col(p, ld, 16 * x, u, lane); }
    __device__ __forceinline__ static int state_row(int x, int g) { return 16 * x + 4 * g; }
    template <int N> __device__ __forceinline__ static void pieces(const f32x4* x, Frag* out) { out[0] = x[0]; }
    typedef f32x4 Tile;                // a score tile's four values of a lane, one per piece
    __device__ __forceinline__ static void put(Tile* p, f32x4 z) { p[0] = z; }
    __device__ __forceinline__ static Frag get(const Tile* p, bool) { return p[0]; }
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
    __device__ __forceinline__ static Frag row(const b16* p, int ld, int r, int u, int g) { return *reinterpret_cast<const bf16x8_t*>(p + r * ld + 32 * u + 8 * g); }
    // transpose reads: 16 lanes read a [4 rows][16 columns] block row-major, each gets the 4 rows of its own column
    __device__ __forceinline__ static s16x4_t tr(const b16* q) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(__attribute__((address_space(3))) const b16*)q); }
    __device__ __forceinline__ static Frag cols(const b16* p, int ld, int u, int lane) {
        const b16* q = p + (32 * u + 4 * (lane >> 4) + ((lane & 15) >> 2)) * ld;
        return __builtin_bit_cast(bf16x8_t, (s16x8_t)__builtin_shufflevector(tr(q), tr(q + 16 * ld), 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ __forceinline__ static Frag col(const b16* p, int ld, int c0, int u, int lane) { return cols(p + c0 + 4 * (lane & 3), ld, u, lane); }
    // the columns of state tile x: tiles 2 y and 2 y + 1 take every other four of 32, so that a lane's rows of both are 8 neighbours, as row() reads them
    __device__ __forceinline__ static Frag state_col(const b16* p, int ld, int x, int u, int lane) {
        return cols(p + 32 * (x >> 1) + 4 * (x & 1) + 8 * (lane & 3), ld, u, lane);
    }
    __device__ __forceinline__ static int state_row(int x, int g) { return 32 * (x >> 1) + 4 * (x & 1) + 8 * g; }
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
    typedef uint2 Tile;
    __device__ __forceinline__ static void put(Tile* p, f32x4 z) {           // pieces 64 places apart
        unsigned a[2], b[2];
        splitn_bf16<2>(z[0], z[1], a);
        splitn_bf16<2>(z[2], z[3], b);
        p[0] = make_uint2(a[0], b[0]);
        p[64] = make_uint2(a[1], b[1]);
    }
    __device__ __forceinline__ static Frag get(const Tile* p, bool two) {    // a tile and the next one
        const uint2 a = p[0];
        uint2 b = make_uint2(0u, 0u);
        if (two) b = p[64 * NS];
        return __builtin_bit_cast(bf16x8_t, u32x4_t{a.x, a.y, b.x, b.y});
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

// z + zeros, NaN if the 16 bytes hold a value that is not finite
template <typename T> __device__ __forceinline__ float probe(u32x4_t r, float z) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned w = r[j];                                     // a value: a cast of the vector's element takes its first one
        if constexpr (sizeof(T) == 4) z = __builtin_fmaf(__uint_as_float(w), 0.f, z);
        else z = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), __builtin_bit_cast(bf16x2_t, 0u), z, false);
    }
    return z;
}

// 16 bytes at any multiple of an element's size
typedef u32x4_t u32x4_a2 __attribute__((aligned(2)));
typedef unsigned u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
// a row of `left` elements, less than 16 bytes of them; zeros behind
template <typename T> __device__ __forceinline__ u32x4_t load_short(const T* p, int left) {
    u32x4_t r = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < (int)(16 / sizeof(T)) - 1; ++j)
        if (j < left) {
            if constexpr (sizeof(T) == 4) r[j] = __float_as_uint(p[j]);
            else r[j >> 1] |= (unsigned)p[j] << (16 * (j & 1));
        }
    return r;
}
// 16 bytes shifted towards the front by n < 128 bits (a multiple of 16, the same for all lanes), zeros behind
__device__ __forceinline__ u32x4_t shift_down(u32x4_t r, int n) {
    if (n & 64) r = u32x4_t{r[2], r[3], 0u, 0u};
    if (n & 32) r = u32x4_t{r[1], r[2], r[3], 0u};
    if (n & 16) r = u32x4_t{r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16, r[3] >> 16};
    return r;
}
__device__ __forceinline__ void store4(float* p, const f32x4& v) { *reinterpret_cast<u32x4_a2*>(p) = __builtin_bit_cast(u32x4_t, v); }
__device__ __forceinline__ void store4(b16* p, const f32x4& v) {
    unsigned a, b, l;
    split2_bf16(v[0], v[1], a, l);
    split2_bf16(v[2], v[3], b, l);
    const u32x2_a2 w = {a, b};
    *reinterpret_cast<u32x2_a2*>(p) = w;
}

// A chunk of one operand: registers on the way from memory to LDS.  WHOLE: rows of whole 16-byte pieces.  Otherwise a row's last piece is read as the
// row's last 16 bytes and shifted on its way to LDS (512 pairs of 1 024 tokens in bf16, 60 x 60: 70 us, 123 element by element; 75 x 75 139, 255; in
// fp32, where three elements at most are read one by one, 368 and 380).
template <typename T, int D, int C, int NT, bool WHOLE> struct Stage {
    static constexpr int E = 16 / sizeof(T), V = D / E, N = C * V / NT, LD = D + Mma<T>::PADK, RS = NT / V;
    static_assert(N * NT == C * V && RS * V == NT, "a chunk is a whole number of pieces per thread, a pass over the threads whole rows");
    u32x4_t r[N];
    // An address is what all threads share (64 bits, in scalar registers: chunk, row pass) plus 32 bits of the thread's own (row of the pass, piece).
    const char* base;            // lowest row of the next chunk's first pass
    unsigned off;
    long pass, chunk;            // bytes from one row pass to the next, and from one chunk
    int row, left, shift;        // first row, elements of it from here on; bits that a last piece moves by; -1: rows of less than 16 bytes
    // rows: token `first` and on in steps of `step` elements (negative from the end; less than 2^22)
    __device__ __forceinline__ void start(const T* first, long step, int dim) {
        row = threadIdx.x / V;
        const int c = threadIdx.x % V * E, low = step < 0 ? RS - 1 - row : row;
        left = dim - c;
        base = (const char*)(first + (step < 0 ? (RS - 1) * step : 0));
        shift = dim < E ? -1 : (E - dim % E) % E * 8 * (int)sizeof(T);
        off = (unsigned)(low * (int)(step < 0 ? -step : step) + (WHOLE || shift < 0 ? c : min(c, dim - E))) * sizeof(T);
        pass = RS * step * (long)sizeof(T);
        chunk = C * step * (long)sizeof(T);
    }
    // the next chunk, of which n rows exist
    __device__ __forceinline__ void load(int n) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const char* p = base + j * pass + off;
            const int have = row + j * RS < n ? left : 0;
            r[j] = u32x4_t{0u, 0u, 0u, 0u};
            if (!WHOLE && shift < 0) r[j] = load_short<T>((const T*)p, have);
            else if (have > 0) r[j] = *reinterpret_cast<const u32x4_a2*>(p);
        }
        base += chunk;
    }
    // Zeros in place of what is not finite; first[c] (in LDS) <- the first row in which column c was that, the chunk's rows counted from `at`
    __device__ __forceinline__ void keep_finite(int* first, int at) {
        float z = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) z = probe<T>(r[j], z);
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(z != z) == 0, 1)) return;
        int me = threadIdx.x;                                        // hidden from the compiler, which would keep this rare path's addresses over all chunks
        asm volatile("" : "+v"(me));
        const int c0 = me % V * E + (!WHOLE && shift > 0 && left < E ? left - E : 0), row0 = at + me / V;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int w = e * (int)sizeof(T) / 4;
                const unsigned mask = sizeof(T) == 4 ? ~0u : 0xffffu << (16 * (e & 1)), top = 0x7f800000u >> (sizeof(T) == 4 || (e & 1) ? 0 : 16);
                if ((r[j][w] & top) == top) {
                    r[j][w] &= ~mask;
                    atomicMin(first + c0 + e, row0 + j * RS);
                }
            }
    }
    __device__ __forceinline__ void store(T* lds) const {
        T* p = lds + threadIdx.x / V * LD + threadIdx.x % V * E;
#pragma unroll
        for (int j = 0; j < N; ++j) *reinterpret_cast<u32x4_t*>(p + j * RS * LD) = !WHOLE && shift > 0 && left < E ? shift_down(r[j], shift) : r[j];
    }
};

// Items of work whose operands come from LDS, each read D items ahead of its use: left alone, the compiler reads every operand right in front of the
// product that waits for it (8 heads of 32 768 tokens in fp32: 75 us, 68 this way).  Vector arithmetic may move between the items, reads and
// products may not.
template <int N, int D, typename Load, typename Use> __device__ __forceinline__ void ahead(Load load, Use use) {
    decltype(load(0)) f[D + 1];
#pragma unroll
    for (int i = 0; i < N + D; ++i) {
        if (i < N) f[i % (D + 1)] = load(i);
        if (i >= D) use(i - D, f[(i - D) % (D + 1)]);
        __builtin_amdgcn_sched_barrier(0x6);
    }
}

__device__ __forceinline__ float decay_power(float g, int n) { return n == 0 ? 1.f : expf(g * (float)n); }
// x e^{g n} as told in front of this file's chunked form; g and n are the same for all lanes, and so are the factor and the choice (in scalar registers)
struct Decay {
    float f;
    int most;                    // of x is kept: f = e^{g n} - 1, otherwise f = e^{g n}
    __device__ __forceinline__ Decay(float g, int n) {
        const float e = g * (float)n;
        most = __builtin_amdgcn_readfirstlane(e > -0.6931472f);
        f = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(most ? expm1f(e) : expf(e))));
    }
    __device__ __forceinline__ float operator()(float x) const { return __builtin_fmaf(x, f, most ? x : 0.f); }
};
__device__ __forceinline__ int row_length(const LinAttnArgs& a, int b) { return a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T; }

// The workgroups of one XCD (every eighth) take neighbouring heads of the same tokens: rows of all heads lie together in memory, and heads that
// share q, k or v find them in that XCD's L2.
__device__ __forceinline__ long xcd_order(long i, long n) { return n % 8 == 0 ? i % 8 * (n / 8) + i / 8 : i; }

// Waves of a workgroup: 16 columns of v each, 32 where Dk and v are both long (or Dk is too short for eight waves to share its rows).  Dk = 64 with
// 128 columns fits 128 registers, so that two workgroups of eight waves run on a compute unit (three rows of up to 5 003 tokens, 12 heads, bf16, the
// call: 70.5 us, 72.5 with four waves; fp32, 16 heads of 8 192 tokens 99.5, 101; bf16 with 512 pairs of 1 024 tokens is better off with four, 110, 105);
// Dk = 128 does not, and eight waves of one workgroup in step with each other are slower than two workgroups of four (512 pairs of 1 024 tokens, before
// the check for NaN: 141 us, 132).  With three waves per SIMD (168 registers, some of them spilled) Dk = Dv = 128 takes 217 us.
constexpr int waves_of(int DKP, int DVP) { return DVP < 64 ? DVP / 16 : (DKP == 64 && DVP == 128 ? 8 : 4); }
constexpr int occupancy_of(int DKP, int DVP) { return waves_of(DKP, DVP) == 8 ? 4 : 2; }
// With Dk > 64 the state takes up to 64 registers of a wave: a chunk half as long leaves room for two waves per SIMD (bf16, 512 pairs of 1 024
// tokens, before the check for NaN: 132 us, 144 with the whole chunk; for Dk <= 64 half a chunk gains 3 % in bf16 and loses 6 % in fp32).
template <typename T> constexpr int chunk_of(int DKP) { return DKP > 64 ? Mma<T>::C / 2 : Mma<T>::C; }

// STATE_ONLY: the segment's own contribution to the state (from zero), nothing is read of q and no o is written.  Two waves per SIMD at least:
// one alone leaves matrix and vector units waiting for each other.
template <typename T, int DKP, int DVP, bool STATE_ONLY, bool WHOLE>
__global__ __launch_bounds__(waves_of(DKP, DVP) * 64, occupancy_of(DKP, DVP)) void linattn_chunk_kernel(const LinAttnArgs a) {
    typedef Mma<T> M;
    constexpr int NW = waves_of(DKP, DVP), NT = NW * 64, DVW = DVP / NW, C = chunk_of<T>(DKP), KB = M::KB, TPF = KB / 16;
    constexpr int KT = DKP / 16, KF = DKP / KB, VT = DVW / 16, CT = C / 16, CF = C / KB;
    constexpr int TILES = CT * (CT + 1) / 2, MINE = (TILES + NW - 1) / NW;      // score tiles of a chunk (s <= t), and of a wave
    const Job& J = a.job[blockIdx.y];
    typedef Stage<T, DKP, C, NT, WHOLE> SK;
    typedef Stage<T, DVP, C, NT, WHOLE> SV;
    __shared__ __attribute__((aligned(16))) T qs[STATE_ONLY ? 8 : C * SK::LD];
    __shared__ __attribute__((aligned(16))) T ks[C * SK::LD];
    __shared__ __attribute__((aligned(16))) T vs[C * SV::LD];
    __shared__ __attribute__((aligned(16))) typename M::Tile ps[STATE_ONLY ? 1 : TILES * M::NS * 64];
    __shared__ int first[STATE_ONLY ? 1 : DVP];                  // a column's first token that is not finite
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4, wave = threadIdx.x >> 6, v0 = wave * DVW;
    if (!STATE_ONLY && lane < DVW) first[v0 + lane] = INT_MAX;
    const long wg = xcd_order(blockIdx.x, gridDim.x);
    const int h = (int)(wg % a.H), seg = (int)(wg / a.H % a.nseg), b = (int)(wg / a.H / a.nseg);
    const long bh = (long)b * a.H + h, D2 = (long)J.Dk * J.Dv;
    const int n = row_length(a, b), beg = seg * a.seg_len, end = min(n, beg + a.seg_len);
    if (STATE_ONLY && beg + a.seg_len >= n) return;             // no token follows: the scan does not read it
    const float g = a.g[h];
    const int e = J.rev ? 0 : 1;
    const long dir = J.rev ? -1 : 1, t0 = J.rev ? n - 1 : 0;     // position p is token t0 + dir p
    const T* q = (const T*)J.q.p + (long)b * J.q.b + (long)(h / J.q.r) * J.q.h + t0 * J.q.t;
    const T* k = (const T*)J.k.p + (long)b * J.k.b + (long)(h / J.k.r) * J.k.h + t0 * J.k.t;
    const T* v = (const T*)J.v.p + (long)b * J.v.b + (long)(h / J.v.r) * J.v.h + t0 * J.v.t;
    const long qt = dir * J.q.t, kt = dir * J.k.t, vt = dir * J.v.t, obase = (long)b * J.ob + (long)h * J.oh;
    const int Dk = J.Dk, Dv = J.Dv;

    SK rq, rk;
    SV rv;
    if (beg < end) {
        if constexpr (!STATE_ONLY) { rq.start(q + beg * qt, qt, Dk); rq.load(end - beg); }
        rk.start(k + beg * kt, kt, Dk);
        rk.load(end - beg);
        rv.start(v + beg * vt, vt, Dv);
        rv.load(end - beg);
    }
    f32x4 S[KT][VT];
    const float* s_in = nullptr;
    int si = J.si, sj = J.sj;
    if constexpr (!STATE_ONLY) {
        if (seg == 0) s_in = J.s_in ? J.s_in + bh * D2 : nullptr;
        else if (beg < n) { s_in = J.seg + (bh * (a.nseg - 1) + seg - 1) * D2; si = J.gi; sj = J.gj; }      // an empty segment computes nothing from it
    }
    const int d_lane = M::state_row(0, grp), j_lane = v0 + col;        // this lane's first element; the others lie at offsets that all lanes share
    const int at_lane = d_lane * si + j_lane * sj;
#pragma unroll
    for (int x = 0; x < KT; ++x)
#pragma unroll
        for (int y = 0; y < VT; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = M::state_row(x, 0) + i, j = 16 * y;
                S[x][y][i] = (s_in && d_lane + d < Dk && j_lane + j < Dv) ? (s_in + (d * si + j * sj))[at_lane] : 0.f;
            }

    // powers of the decay: between the tokens of this wave's score tiles (nothing where s > t), in front of a tile of tokens, to the chunk's end
    float pw[MINE][4], pin[CT], wst[CF][KB / 4];
    int tx[MINE], ts[MINE];
    unsigned past = 0;                                              // a token to come counts as nothing, whatever its score (0 * inf is not 0)
    if constexpr (!STATE_ONLY) {
#pragma unroll
        for (int m = 0; m < MINE; ++m) {
            const int id = wave + m * NW;
            tx[m] = (id >= 1) + (id >= 3) + (id >= 6);
            ts[m] = id - tx[m] * (tx[m] + 1) / 2;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 16 * (tx[m] - ts[m]) + col - M::srow(grp, i);
                pw[m][i] = J.uscale * J.oscale * decay_power(g, max(0, d));
                past |= (unsigned)(d >= 0) << (4 * m + i);
            }
        }
    }
    float pt[CT];                                                    // whole tiles of tokens
#pragma unroll
    for (int x = 0; x < CT; ++x) pt[x] = decay_power(g, 16 * x);
    if constexpr (!STATE_ONLY) {
        const float p0 = J.oscale * decay_power(g, col + e);
#pragma unroll
        for (int x = 0; x < CT; ++x) pin[x] = p0 * pt[x];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p0 = J.uscale * decay_power(g, 16 - e - M::srow(grp, i));
#pragma unroll
        for (int x = 0; x < CT; ++x) wst[x / TPF][4 * (x % TPF) + i] = p0 * pt[CT - 1 - x];
    }
    Decay fade(g, C);

    // o likewise: the lowest row of 16 tokens, and this lane's place from there
    const int osize = J.o16 ? 2 : 4;
    const long ostep = dir * J.ot * osize;
    char* obase16 = (char*)J.o + (obase + (t0 + dir * beg + (J.rev ? -15 : 0)) * J.ot) * osize;
    const unsigned olane = (unsigned)((J.rev ? 15 - col : col) * (int)J.ot + v0 + 4 * grp) * osize;
    for (int c0 = beg; c0 < end; c0 += C, obase16 += C * ostep) {
        __syncthreads();
        if constexpr (!STATE_ONLY) rq.store(qs);
        rk.store(ks);
        // A score of 0 does not keep NaN or infinity in v from the tokens in front of it.  The products take 0 for them, and behind the last chunk what a
        // column's first one reaches is made NaN.  (1 % of a call; looking at the state at a segment's end and doing it again where one is there 2 to 3 %, a
        // second pass costs the first its registers.)
        if constexpr (!STATE_ONLY) rv.keep_finite(first, c0);
        rv.store(vs);
        __syncthreads();
        const int L = min(C, end - c0), c1 = c0 + C;
        if (c1 < end) {
            if constexpr (!STATE_ONLY) rq.load(end - c1);
            rk.load(end - c1);
            rv.load(end - c1);
        }
        typename M::Frag vf[CF][VT];
#pragma unroll
        for (int u = 0; u < CF; ++u)
#pragma unroll
            for (int y = 0; y < VT; ++y) vf[u][y] = M::col(vs, SV::LD, v0 + 16 * y, u, lane);
        if constexpr (!STATE_ONLY) {
            // this wave's score tiles, for all
#pragma unroll
            for (int m = 0; m < MINE; ++m)
                if (wave + m * NW < TILES) {
                    f32x4 z = {0.f, 0.f, 0.f, 0.f};
                    struct Pair { typename M::Frag k, q; };
                    ahead<KF, KF>([&](int w) { return Pair{M::row(ks, SK::LD, 16 * ts[m] + M::krow(col), w, grp), M::row(qs, SK::LD, 16 * tx[m] + col, w, grp)}; },
                                  [&](int, const Pair& f) { z = M::mma(f.k, f.q, z); });
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[i] = past >> (4 * m + i) & 1 ? z[i] * pw[m][i] : 0.f;
                    M::put(ps + (wave + m * NW) * (M::NS * 64) + lane, z);
                }
            f32x4 acc[CT][VT];
#pragma unroll
            for (int x = 0; x < CT; ++x)
#pragma unroll
                for (int y = 0; y < VT; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
            // q S
            typename M::Frag sf[VT][M::NS];
            ahead<KF * CT, 2>([&](int i) { return M::row(qs, SK::LD, 16 * (i % CT) + col, i / CT, grp); },
                              [&](int i, const typename M::Frag& qf) {
                const int x = i % CT, u = i / CT;
                if (x == 0)
#pragma unroll
                    for (int y = 0; y < VT; ++y) {
                        f32x4 t[TPF];
#pragma unroll
                        for (int p = 0; p < TPF; ++p) t[p] = S[u * TPF + p][y];
                        M::template pieces<M::NS>(t, sf[y]);
                    }
#pragma unroll
                for (int p = M::NS - 1; p >= 0; --p)
#pragma unroll
                    for (int y = 0; y < VT; ++y) acc[x][y] = M::mma(sf[y][p], qf, acc[x][y]);
            });
#pragma unroll
            for (int x = 0; x < CT; ++x)
#pragma unroll
                for (int y = 0; y < VT; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[x][y][i] *= pin[x];
            __syncthreads();                                     // the scores are there
#pragma unroll
            for (int x = 0; x < CT; ++x) {
#pragma unroll
                for (int u = 0; u * TPF <= x; ++u) {
                    const typename M::Tile* t = ps + (x * (x + 1) / 2 + u * TPF) * (M::NS * 64) + lane;
                    typename M::Frag pf[M::NS];
#pragma unroll
                    for (int p = 0; p < M::NS; ++p) pf[p] = M::get(t + 64 * p, u * TPF + 1 <= x);
#pragma unroll
                    for (int p = M::NS - 1; p >= 0; --p)
#pragma unroll
                        for (int y = 0; y < VT; ++y) acc[x][y] = M::mma(vf[u][y], pf[p], acc[x][y]);
                }
                const int r = 16 * x + col;
                if (r < L) {
                    char* const row = obase16 + 16 * x * ostep;
#pragma unroll
                    for (int y = 0; y < VT; ++y) {
                        const int j = v0 + 16 * y + 4 * grp;
                        if (j >= Dv) continue;
                        char* const at = row + 16 * y * osize + olane;
                        if (WHOLE || j + 4 <= Dv) {
                            if (J.o16) store4((b16*)at, acc[x][y]); else store4((float*)at, acc[x][y]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 3; ++i)
                                if (j + i < Dv) { if (J.o16) st1((b16*)at, i, acc[x][y][i]); else st1((float*)at, i, acc[x][y][i]); }
                        }
                    }
                }
            }
        }
        // the state
        if (L < C) {                                               // the last chunk of a row
#pragma unroll
            for (int u = 0; u < CF; ++u)
#pragma unroll
                for (int j = 0; j < KB / 4; ++j)
                    wst[u][j] = J.uscale * decay_power(g, max(0, L - e - (KB * u + 16 * (j >> 2) + M::srow(grp, j & 3))));
            fade = Decay(g, L);
        }
        if (fade.most) {
#pragma unroll
            for (int x = 0; x < KT; ++x)
#pragma unroll
                for (int y = 0; y < VT; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[x][y][i] = __builtin_fmaf(S[x][y][i], fade.f, S[x][y][i]);
        } else {
#pragma unroll
            for (int x = 0; x < KT; ++x)
#pragma unroll
                for (int y = 0; y < VT; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[x][y][i] *= fade.f;
        }
        typename M::Frag wf[VT][M::NV];
        ahead<CF * KT, 2>([&](int i) { return M::state_col(ks, SK::LD, i % KT, i / KT, lane); },
                          [&](int i, const typename M::Frag& kf) {
            const int x = i % KT, u = i / KT;
            if (x == 0)
#pragma unroll
                for (int y = 0; y < VT; ++y) {
                    f32x4 t[TPF];
                    M::scaled(vf[u][y], wst[u], t);
                    M::template pieces<M::NV>(t, wf[y]);
                }
#pragma unroll
            for (int p = M::NV - 1; p >= 0; --p)
#pragma unroll
                for (int y = 0; y < VT; ++y) S[x][y] = M::mma(kf, wf[y][p], S[x][y]);
        });
    }
    if constexpr (!STATE_ONLY) {
        // from a column's first value on that is not finite: the outputs, behind those that other lanes stored there, and the state
        const int f = lane < DVW ? first[v0 + lane] : INT_MAX;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(f != INT_MAX) != 0, 0)) {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
            __builtin_amdgcn_s_waitcnt(0);
            const int j = v0 + lane % DVW, from = first[j];
            if (from != INT_MAX && j < Dv)
                for (int c = from + lane / DVW; c < end; c += 64 / DVW) {
                    char* const p = (char*)J.o + (obase + (t0 + dir * c) * J.ot + j) * osize;
                    if (J.o16) st1((b16*)p, 0, __builtin_nanf("")); else st1((float*)p, 0, __builtin_nanf(""));
                }
#pragma unroll
            for (int y = 0; y < VT; ++y)
                if (first[j_lane + 16 * y] != INT_MAX)
#pragma unroll
                    for (int x = 0; x < KT; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) S[x][y][i] = __builtin_nanf("");
        }
    }
    float* s_out;
    int oi = J.si, oj = J.sj;
    if constexpr (STATE_ONLY) {
        s_out = J.seg + (bh * (a.nseg - 1) + seg) * D2;
        oi = J.gi; oj = J.gj;
    } else {
        // behind the row's last token: o is zero
        const int z0 = max(n, beg), zn = max(0, min(a.T, beg + a.seg_len) - z0);
        for (long x = threadIdx.x; x < (long)zn * Dv; x += NT) {
            const long at = obase + (z0 + x / Dv) * J.ot + x % Dv;
            if (J.o16) ((b16*)J.o)[at] = 0; else ((float*)J.o)[at] = 0.f;
        }
        if (!J.s_out || seg != (n > 0 ? (n - 1) / a.seg_len : 0)) return;      // the segment with the row's last token
        s_out = J.s_out + bh * D2;
    }
    const int out_lane = d_lane * oi + j_lane * oj;
#pragma unroll
    for (int x = 0; x < KT; ++x)
#pragma unroll
        for (int y = 0; y < VT; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = M::state_row(x, 0) + i, j = 16 * y;
                if (d_lane + d < Dk && j_lane + j < Dv) (s_out + (d * oi + j * oj))[out_lane] = S[x][y][i];
            }
}

// seg[i] <- the state behind segment i: one thread per element, the segments' own contributions loaded eight at a time (8 pairs of 64 states of
// 64 x 64: 10.5 us, the latency of eight such rounds; 36 pairs of 15 states of 64 x 128: 7 us)
__global__ __launch_bounds__(256) void linattn_segment_scan_kernel(const LinAttnArgs a) {
    const Job& J = a.job[0];
    const int x = blockIdx.y * 256 + threadIdx.x, D = J.Dk * J.Dv, bh = blockIdx.x;
    if (x >= D) return;
    const int n = row_length(a, bh / a.H);
    const float g = a.g[bh % a.H];
    float* p = J.seg + (long)bh * (a.nseg - 1) * D + x;
    float run = J.s_in ? J.s_in[(long)bh * D + x] : 0.f;
    const Decay fade(g, a.seg_len);
    for (int i0 = 0; i0 < a.nseg - 1; i0 += 8) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (i0 + i < a.nseg - 1 && (long)(i0 + i + 1) * a.seg_len < n) ? p[(long)(i0 + i) * D] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i0 + i >= a.nseg - 1 || (long)(i0 + i + 1) * a.seg_len >= n) return;      // what follows enters no token's segment
            run = fade(run) + y[i];
            p[(long)(i0 + i) * D] = run;
        }
    }
}

// One token: a block per (batch row, head), bound by the state's one read and one write.  The decay is that of the chunked form: a factor rounded to
// fp32 would let a long stream drift from the same prompt (5e-4 after 16 384 tokens at 1 - 2^-12).  Thread = (row group, V neighbouring columns), eight
// rows in flight each; the partial sums over the row groups meet in LDS.  256 rows of 16 heads, 128 x 128: 105 us = 5.1 TB/s (a large copy: 4.9); one row
// of 5 heads, 60 x 60: 3.9 us, the launch.
template <typename T, int V>
__global__ __launch_bounds__(256) void linattn_step_kernel(const LinAttnArgs a, int lpr /* threads per row, a power of two with lpr * V >= Dv */) {
    __shared__ float qs[128], ks[128], red[256 * V];
    const Job& J = a.job[0];
    const int h = blockIdx.x % a.H, b = blockIdx.x / a.H, tid = threadIdx.x, Dk = J.Dk, Dv = J.Dv;
    const T* q = (const T*)J.q.p + (long)b * J.q.b + (long)(h / J.q.r) * J.q.h;
    const T* k = (const T*)J.k.p + (long)b * J.k.b + (long)(h / J.k.r) * J.k.h;
    const T* v = (const T*)J.v.p + (long)b * J.v.b + (long)(h / J.v.r) * J.v.h;
    const int j = tid % lpr * V, r0 = tid / lpr, groups = 256 / lpr;
    float* S = J.s_out + ((long)b * a.H + h) * Dk * Dv + j;
    float vv[V], acc[V];
#pragma unroll
    for (int c = 0; c < V; ++c) { vv[c] = j < Dv ? ld1(v, j + c) : 0.f; acc[c] = 0.f; }
    if (tid < Dk) { qs[tid] = ld1(q, tid); ks[tid] = ld1(k, tid); }
    __syncthreads();
    const Decay fade(a.g[h], 1);
    if (j < Dv)
        for (int d0 = r0; d0 < Dk; d0 += 8 * groups) {
            float s[8][V];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int d = d0 + u * groups;
                if (d < Dk) {
                    if constexpr (V == 4) { const float4 x = ld4(S + (long)d * Dv, 0); s[u][0] = x.x; s[u][1] = x.y; s[u][2] = x.z; s[u][3] = x.w; }
                    else s[u][0] = S[(long)d * Dv];
                }
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int d = d0 + u * groups;
                if (d < Dk) {
#pragma unroll
                    for (int c = 0; c < V; ++c) { s[u][c] = fade(s[u][c]) + ks[d] * vv[c]; acc[c] += qs[d] * s[u][c]; }
                    if constexpr (V == 4) st4(S + (long)d * Dv, 0, make_float4(s[u][0], s[u][1], s[u][2], s[u][3]));
                    else S[(long)d * Dv] = s[u][0];
                }
            }
        }
#pragma unroll
    for (int c = 0; c < V; ++c) red[tid * V + c] = acc[c];
    __syncthreads();
    if (tid < Dv) {
        float s = 0.f;
        for (int r = 0; r < groups; ++r) s += red[r * lpr * V + tid];
        st1((T*)J.o + (long)b * J.ob + (long)h * J.oh, tid, s * J.oscale);
    }
}

// out[r][c] = sum over j < n of x[r][c / D][j][c % D]: the gradient of a head that n heads read, in the order of the heads.  Bound by memory:
// 16 384 tokens of 16 heads of 128 into 4, 151 MB: 22 us (6.8 TB/s, much of it from the last-level cache the products just wrote)
template <typename T, int V>
__global__ __launch_bounds__(256) void head_sum_kernel(const float* __restrict__ x, T* __restrict__ out, long rows, int n, int D) {
    const long total = rows * (D / V);                    // rows: one per token and shared head
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long r = i / (D / V);
        const int d = (int)(i - r * (D / V)) * V;
        const float* p = x + r * n * D + d;
        if constexpr (V == 4) {
            float4 s = ld4(p, 0);
            for (int j = 1; j < n; ++j) { const float4 y = ld4(p + (long)j * D, 0); s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w; }
            st4(out + r * D + d, 0, s);
        } else {
            float s = p[0];
            for (int j = 1; j < n; ++j) s += p[(long)j * D];
            st1(out, r * D + d, s);
        }
    }
}

// Segments of the time axis: one pass over q, k, v where the rows and heads alone give every compute unit half of the eight waves it should have;
// otherwise the axis is split so that the eight are there, at no less than two chunks a segment, for a second read of k and v and the segments'
// states.  With sixteen waves the scan over the states grows by more than the chunks save (8 heads of 32 768 tokens: scan 20 us, 10.7; chunks 74, 70;
// three ragged prompts 79 us, 69; 60 calls drawn from all sizes, geometric mean: 46.0 us, 45.0).
void segments(int B, int T, int H, int Dv, int b16_io, int* nseg, int* len) {
    const int C = b16_io ? Mma<b16>::C : Mma<float>::C, chunks = (int)(((long)T + C - 1) / C), groups = hw_cu_count() * (Dv <= 32 ? 4 : 2);
    const long rows = (long)B * H;
    long want = 2 * rows >= groups || rows < 1 ? 1 : (groups + rows - 1) / rows;
    if (want > chunks / 2) want = chunks / 2;
    if (want < 1) want = 1;
    const int per = chunks > 0 ? (int)((chunks + want - 1) / want) : 1;
    *nseg = chunks > 0 ? (chunks + per - 1) / per : 1;
    *len = per * C;
}

template <typename T, int DKP, int DVP> void chunk_launch(const LinAttnArgs& a, int jobs, bool state_only, hipStream_t st) {
    const dim3 grid((unsigned)((long)a.B * a.H * a.nseg), jobs), block(waves_of(DKP, DVP) * 64);
    const int piece = 16 / (int)sizeof(T);
    bool whole = true;                   // rows of whole 16-byte pieces
    for (int j = 0; j < jobs; ++j) whole = whole && a.job[j].Dk % piece == 0 && a.job[j].Dv % piece == 0;
    if (state_only) {
        if (whole) hipLaunchKernelGGL((linattn_chunk_kernel<T, DKP, DVP, true, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((linattn_chunk_kernel<T, DKP, DVP, true, false>), grid, block, 0, st, a);
    } else {
        if (whole) hipLaunchKernelGGL((linattn_chunk_kernel<T, DKP, DVP, false, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((linattn_chunk_kernel<T, DKP, DVP, false, false>), grid, block, 0, st, a);
    }
}
template <typename T, int DKP> void chunk_launch_v(const LinAttnArgs& a, int jobs, bool state_only, hipStream_t st) {
    if (a.job[0].Dv <= 32) chunk_launch<T, DKP, 32>(a, jobs, state_only, st);
    else if (a.job[0].Dv <= 64) chunk_launch<T, DKP, 64>(a, jobs, state_only, st);
    else chunk_launch<T, DKP, 128>(a, jobs, state_only, st);
}
template <typename T> void chunk_launch_k(const LinAttnArgs& a, int jobs, bool state_only, hipStream_t st) {
    if (a.job[0].Dk <= 32) chunk_launch_v<T, 32>(a, jobs, state_only, st);
    else if (a.job[0].Dk <= 64) chunk_launch_v<T, 64>(a, jobs, state_only, st);
    else chunk_launch_v<T, 128>(a, jobs, state_only, st);
}
// jobs of one size of Dk and Dv (up to their tiles) share a launch
int run_chunks(const LinAttnArgs& a, int jobs, bool state_only, int b16_io, hipStream_t st) {
    if (b16_io) chunk_launch_k<b16>(a, jobs, state_only, st);
    else chunk_launch_k<float>(a, jobs, state_only, st);
    HA2G_CHECK_LAUNCH("linattn");
    return 0;
}
int run_scan(const LinAttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(linattn_segment_scan_kernel, dim3(a.B * a.H, (a.job[0].Dk * a.job[0].Dv + 255) / 256), dim3(256), 0, st, a);
    HA2G_CHECK_LAUNCH("linattn: segments");
    return 0;
}
int tile_of(int d) { return d <= 32 ? 32 : (d <= 64 ? 64 : 128); }

constexpr long STRIDE_LIMIT = 1L << 22;      // of a token, in elements: a workgroup's rows lie within 32 bits of each other
// one token has no next one: its stride may be anything
int check_strides(const char* what, const long* strides, int n, int T) {
    HA2G_REQUIRE(strides, "%s: null strides", what);
    for (int i = 1; T > 1 && i < 3 * n; i += 3)
        HA2G_REQUIRE(strides[i] >= 0 && strides[i] < STRIDE_LIMIT, "%s: a token stride of %ld elements (0 to %ld)", what, strides[i], STRIDE_LIMIT - 1);
    return 0;
}
long token_stride(const long* s, int T) { return T > 1 ? s[1] : 0; }

Operand operand(const void* p, const long* s, int r, int T) { return {p, s[0], token_stride(s, T), s[2], r}; }

void set_out(Job& j, void* o, const long* s, int o16, int T) {
    j.o = o; j.ob = s[0]; j.ot = token_stride(s, T); j.oh = s[2]; j.o16 = o16;
}
// one segment's worth of states lies as the forward pass has it, [Dk][Dv]; `turned` where the job's state is that transposed
void set_state(Job& j, const float* s_in, float* s_out, float* seg, bool turned) {
    j.s_in = s_in; j.s_out = s_out; j.seg = seg;
    j.si = j.gi = turned ? 1 : j.Dv;
    j.sj = j.gj = turned ? j.Dk : 1;
}

int check_args(LinAttnArgs& a, const char* what, const float* g, const int* lengths, int B, int T, int H, int rq, int rk, int rv, int Dk, int Dv, int b16_io,
               bool operands) {
    HA2G_REQUIRE(B >= 0 && T >= 0 && H >= 1 && Dk >= 1 && Dk <= 128 && Dv >= 1 && Dv <= 128, "%s: B=%d T=%d H=%d Dk=%d Dv=%d (1 <= Dk, Dv <= 128)", what, B,
                 T, H, Dk, Dv);
    HA2G_REQUIRE(rq >= 1 && rk >= 1 && rv >= 1 && H % rq == 0 && H % rk == 0 && H % rv == 0, "%s: %d heads shared by %d / %d / %d", what, H, rq, rk, rv);
    HA2G_REQUIRE(B == 0 || (g && (T == 0 || operands)), "%s: null operand", what);
    a.g = g; a.lengths = lengths; a.B = B; a.T = T; a.H = H;
    segments(B, T, H, Dv, b16_io, &a.nseg, &a.seg_len);
    HA2G_REQUIRE((long)B * H * a.nseg < 1L << 23, "%s: B * H * segments = %ld (a grid has less than 2^32 threads)", what, (long)B * H * a.nseg);
    HA2G_REQUIRE((long)T + a.seg_len <= 0x7fffffffL, "%s: T = %d", what, T);
    return 0;
}

}  // namespace

extern "C" {

long ha2g_linattn_workspace_floats(int B, int T, int H, int Dk, int Dv, int b16_io) {
    int nseg, len;
    if (B < 1 || H < 1 || T < 1) return 0;
    segments(B, T, H, Dv, b16_io, &nseg, &len);
    return (long)B * H * (nseg - 1) * Dk * Dv;
}

int ha2g_linattn_fwd(const void* q, const void* k, const void* v, void* o, const float* log_decay, const float* s_in, float* s_out, const int* lengths,
                     const long* strides, int B, int T, int H, int rq, int rk, int rv, int Dk, int Dv, float scale, int b16_io, float* ws, void* stream) {
    LinAttnArgs a;
    if (const int rc = check_args(a, "linattn_fwd", log_decay, lengths, B, T, H, rq, rk, rv, Dk, Dv, b16_io, q && k && v && o)) return rc;
    if (B == 0) return 0;
    if (const int rc = check_strides("linattn_fwd", strides, 4, T)) return rc;
    HA2G_REQUIRE(a.nseg == 1 || ws, "linattn_fwd: no workspace (ha2g_linattn_workspace_floats)");
    Job& j = a.job[0];
    j.q = operand(q, strides, rq, T); j.k = operand(k, strides + 3, rk, T); j.v = operand(v, strides + 6, rv, T);
    j.Dk = Dk; j.Dv = Dv; j.rev = 0; j.oscale = scale; j.uscale = 1.f;
    set_out(j, o, strides + 9, b16_io, T);
    set_state(j, s_in, s_out, ws, false);
    const hipStream_t st = (hipStream_t)stream;
    if (a.nseg > 1) {
        if (const int rc = run_chunks(a, 1, true, b16_io, st)) return rc;
        if (const int rc = run_scan(a, st)) return rc;
    }
    return run_chunks(a, 1, false, b16_io, st);
}

int ha2g_linattn_bwd(const void* q, const void* k, const void* v, const void* dout, void* dq, void* dk, void* dv, const float* log_decay, const float* s_in,
                     const float* ds_out, float* ds_in, const int* lengths, const long* strides, int B, int T, int H, int rq, int rk, int rv, int Dk, int Dv,
                     float scale, int b16_io, int dq_b16, int dk_b16, int dv_b16, const float* ws_fwd, float* ws, void* stream) {
    LinAttnArgs a;
    if (const int rc = check_args(a, "linattn_bwd", log_decay, lengths, B, T, H, rq, rk, rv, Dk, Dv, b16_io, q && k && v && dout)) return rc;
    HA2G_REQUIRE(B == 0 || dv || !ds_in || T == 0, "linattn_bwd: the gradient of the first state comes with dv");
    if (B == 0) return 0;
    if (const int rc = check_strides("linattn_bwd", strides, 7, T)) return rc;
    HA2G_REQUIRE(a.nseg == 1 || (ws && (ws_fwd || !dq)), "linattn_bwd: no workspace (ha2g_linattn_workspace_floats)");
    const Operand oq_ = operand(q, strides, rq, T), ok_ = operand(k, strides + 3, rk, T), ov_ = operand(v, strides + 6, rv, T),
                  od_ = operand(dout, strides + 9, 1, T);
    Job jv, jk, jq;
    jv.q = ok_; jv.k = oq_; jv.v = od_; jv.Dk = Dk; jv.Dv = Dv; jv.rev = 1; jv.oscale = 1.f; jv.uscale = scale;
    set_out(jv, dv, strides + 18, dv_b16, T);
    set_state(jv, ds_out, ds_in, ws, false);
    jk.q = ov_; jk.k = od_; jk.v = oq_; jk.Dk = Dv; jk.Dv = Dk; jk.rev = 1; jk.oscale = 1.f; jk.uscale = scale;
    set_out(jk, dk, strides + 15, dk_b16, T);
    set_state(jk, ds_out, nullptr, ws, true);
    jq.q = od_; jq.k = ov_; jq.v = ok_; jq.Dk = Dv; jq.Dv = Dk; jq.rev = 0; jq.oscale = scale; jq.uscale = 1.f;
    set_out(jq, dq, strides + 12, dq_b16, T);
    set_state(jq, s_in, nullptr, const_cast<float*>(ws_fwd), true);
    const hipStream_t st = (hipStream_t)stream;
    if (a.nseg > 1 && (dv || dk)) {                      // both walk through the same states; dq through the forward pass's
        a.job[0] = jv;
        if (const int rc = run_chunks(a, 1, true, b16_io, st)) return rc;
        if (const int rc = run_scan(a, st)) return rc;
    }
    const bool same = tile_of(Dk) == tile_of(Dv);
    int n = 0;
    if (dv || ds_in) a.job[n++] = jv;
    if (!same && n) {
        if (const int rc = run_chunks(a, n, false, b16_io, st)) return rc;
        n = 0;
    }
    if (dk) a.job[n++] = jk;
    if (dq) a.job[n++] = jq;
    return n ? run_chunks(a, n, false, b16_io, st) : 0;
}

int ha2g_linattn_step(const void* q, const void* k, const void* v, void* o, const float* log_decay, float* state, const long* strides, int B, int H,
                      int rq, int rk, int rv, int Dk, int Dv, float scale, int b16_io, void* stream) {
    LinAttnArgs a;
    if (const int rc = check_args(a, "linattn_step", log_decay, nullptr, B, 1, H, rq, rk, rv, Dk, Dv, b16_io, q && k && v && o && state)) return rc;
    if (B == 0) return 0;
    if (const int rc = check_strides("linattn_step", strides, 4, 1)) return rc;
    Job& j = a.job[0];
    j.q = operand(q, strides, rq, 1); j.k = operand(k, strides + 3, rk, 1); j.v = operand(v, strides + 6, rv, 1);
    j.Dk = Dk; j.Dv = Dv; j.oscale = scale;
    set_out(j, o, strides + 9, b16_io, 1);
    j.s_out = state;
    const bool wide = Dv % 4 == 0 && (uintptr_t)state % 16 == 0;
    int lpr = 1;
    while (lpr * (wide ? 4 : 1) < Dv) lpr *= 2;
    const dim3 grid(B * H), block(256);
    if (b16_io && wide) hipLaunchKernelGGL((linattn_step_kernel<b16, 4>), grid, block, 0, (hipStream_t)stream, a, lpr);
    else if (b16_io) hipLaunchKernelGGL((linattn_step_kernel<b16, 1>), grid, block, 0, (hipStream_t)stream, a, lpr);
    else if (wide) hipLaunchKernelGGL((linattn_step_kernel<float, 4>), grid, block, 0, (hipStream_t)stream, a, lpr);
    else hipLaunchKernelGGL((linattn_step_kernel<float, 1>), grid, block, 0, (hipStream_t)stream, a, lpr);
    HA2G_CHECK_LAUNCH("linattn_step");
    return 0;
}

int ha2g_head_sum(const float* x, void* out, long rows, int heads, int n, int D, int b16_out, void* stream) {
    HA2G_REQUIRE(rows >= 0 && heads >= 1 && n >= 1 && D >= 1, "head_sum: rows=%ld heads=%d n=%d D=%d", rows, heads, n, D);
    if (rows == 0) return 0;
    HA2G_REQUIRE(x && out, "head_sum: null operand");
    const bool wide = D % 4 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)out % (b16_out ? 8 : 16) == 0;
    const long want = (rows * heads * (wide ? D / 4 : D) + 255) / 256;
    const dim3 grid((unsigned)(want > 16384 ? 16384 : want)), block(256);
    const hipStream_t st = (hipStream_t)stream;
    if (b16_out && wide) hipLaunchKernelGGL((head_sum_kernel<b16, 4>), grid, block, 0, st, x, (b16*)out, rows * heads, n, D);
    else if (b16_out) hipLaunchKernelGGL((head_sum_kernel<b16, 1>), grid, block, 0, st, x, (b16*)out, rows * heads, n, D);
    else if (wide) hipLaunchKernelGGL((head_sum_kernel<float, 4>), grid, block, 0, st, x, (float*)out, rows * heads, n, D);
    else hipLaunchKernelGGL((head_sum_kernel<float, 1>), grid, block, 0, st, x, (float*)out, rows * heads, n, D);
    HA2G_CHECK_LAUNCH("head_sum");
    return 0;
}

}  // extern "C"
