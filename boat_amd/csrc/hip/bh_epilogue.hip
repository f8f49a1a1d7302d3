// bh_epilogue.hip - a matrix product whose stores finish the layer: C = act(op(A).op(B) + bias) + residual.
//
// A dense layer of a transformer is z = x.W + b, y = act(z), and often h = y + residual (src/layers/dense.c:135-188 and the
// elementwise passes behind it).  Each pass behind the product reads and writes the whole [rows, features] matrix; here the
// accumulators go through bias, activation and residual in registers, and what the backward pass needs (z, or act(z) for the
// activations whose derivative is a function of it) is stored beside the result.
//
// The products run on the bf16 matrix cores from operands split into three bf16 each (bh_split.h): fp32 sums at six bf16
// instructions per product, 2.7 times the rate of the fp32 matrix instruction.
#include "bh_split.h"

#include <math.h>

#include <type_traits>

namespace bh {

struct EpiArgs {
    const float* a; const float* b;
    int64_t m, n, k, lda, ldb;
    float* c; int64_t ldc;
    const float* bias;                       // [n] or NULL
    float* saved; int64_t lds;               // [m, n] or NULL
    const float* residual; int64_t ldr;      // [m, n] or NULL; may be c itself
    int act;
    int tiles_m, tiles_n;
    int splits;                              // > 1: partial sums go to `partial` [split][m][n], epilogue_fold_kernel finishes
    int64_t k_per_split;                     // multiple of 16
    float* partial;
    float* colsum; int colsum_add;           // small tiles, both operands along rows: [n] (+)= column sums of B, or NULL
};

// erf as GELU needs it, without a branch: 1 - erf(t) = 2^(-t P(t)), P the polynomial of degree 8 whose largest error in erf over
// [0, 4] is least (by linear programming); from 4 on erf is 1 in fp32.  Evaluated in fp32 it is off by at most 9.1e-8, and the
// hardware exponential adds up to one step of [1/2, 1): 1.5e-7 absolute, where 1 + erf rounds to 6e-8.  The GELU of a dense sweep
// of [-6, 6] is off by at most 1.13e-7 |z| (1.22e-7 with erff), next to zero by 7.7e-8 |z| (6.2e-8).
// 8192 x 4096 over 1024 with GELU and z kept 335 us, 349 with erff, 330 without an activation.
__device__ __forceinline__ float erf_absolute(float x) {
    const float t = fminf(fabsf(x), 4.f);
    float p = -1.1604582e-05f;
    p = fmaf(p, t, 1.529623e-04f);
    p = fmaf(p, t, -8.482268e-04f);
    p = fmaf(p, t, 2.2747705e-03f);
    p = fmaf(p, t, -8.478805e-05f);
    p = fmaf(p, t, -2.7724488e-02f);
    p = fmaf(p, t, 1.4830792e-01f);
    p = fmaf(p, t, 9.184429e-01f);
    p = fmaf(p, t, 1.6279073f);
    return copysignf(1.f - __builtin_amdgcn_exp2f(-(p * t)), x);
}

__device__ __forceinline__ float act_value(int act, float z) {
    switch (act) {
        case BH_ACT_RELU: return z > 0.f || z != z ? z : 0.f;
        case BH_ACT_SIGMOID: return 1.f / (1.f + expf(-z));
        case BH_ACT_TANH: return tanhf(z);
        case BH_ACT_GELU: return z * (0.5f * (1.f + erf_absolute(z * 0.70710678118654752440f)));
    }
    return z;
}
// what bh_activation_backward reads: the input of ReLU and GELU, the output of sigmoid and tanh
__device__ __forceinline__ bool saves_output(int act) { return act == BH_ACT_SIGMOID || act == BH_ACT_TANH; }

__device__ __forceinline__ bool finite_f32(float v) { return fabsf(v) <= 3.402823466e38f; }

// One element of the product in plain fp32 arithmetic: for sums the split could not carry (infinities, NaN).  Eight of the
// contraction are on their way at a time, and a sum that has become NaN stays one.  8192 x 4096 over 1024, every element not
// finite: 0.58 ms where they are NaN (a diverged step; 0.34 without), 32 ms where they are infinities.
template <bool A_KC, bool B_KC>
__device__ __forceinline__ float plain_element(const EpiArgs& g, int64_t row, int64_t col, int64_t k0, int64_t k1) {
    constexpr int kAhead = 8;
    const float* a = g.a + (A_KC ? row * g.lda : row);
    const float* b = g.b + (B_KC ? col * g.ldb : col);
    float s = 0.f;
    for (int64_t k = k0; k < k1 && s == s; k += kAhead) {
        float x[kAhead], y[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; e++) {
            const bool there = k + e < k1;
            x[e] = there ? a[A_KC ? k + e : (k + e) * g.lda] : 0.f;
            y[e] = there ? b[B_KC ? k + e : (k + e) * g.ldb] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < kAhead; e++) s = fmaf(x[e], y[e], s);
    }
    return s;
}

__device__ __forceinline__ void finish_element(const EpiArgs& g, int64_t row, int64_t col, float sum) {
    float z = sum + (g.bias ? g.bias[col] : 0.f);
    float y = act_value(g.act, z);
    if (g.saved) g.saved[row * g.lds + col] = saves_output(g.act) ? y : z;
    if (g.residual) y += g.residual[row * g.ldr + col];
    g.c[row * g.ldc + col] = y;
}

// workgroup number -> output tile: neighbours in launch order go to different XCDs, so each XCD gets a contiguous run of
// tiles (its own L2), walked in groups of 8 tile rows
__device__ __forceinline__ void tile_of(int pid, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int total = tiles_m * tiles_n;
    if (total % kNumXcd == 0) pid = (pid % kNumXcd) * (total / kNumXcd) + pid / kNumXcd;
    constexpr int kGroup = 8;
    const int per = kGroup * tiles_n, first = pid / per * kGroup;
    const int rows = min(tiles_m - first, kGroup);
    tm = first + pid % per % rows;
    tn = pid % per / rows;
}

// ---------------------------------------------------------------------------------------------------- finishing a tile
// A wavefront's finished 32 x (32*TN) block of sums goes through LDS (rows padded by 8 floats), so that the rest runs over
// whole rows: 16-byte loads and stores, one copy of the activation's code, and the rare recomputation can index its element.
template <int TN> struct EpiBlock {
    static constexpr int LD = 32 * TN + 8;       // floats
    static constexpr int BYTES = 32 * LD * (int)sizeof(float);
};

template <int TN, bool A_KC, bool B_KC>
__device__ __forceinline__ void finish_block(const EpiArgs& g, const f32x16 (&acc)[TN], float* lds, int64_t row0, int64_t col0, int lane,
                                             bool vec) {
    constexpr int LD = EpiBlock<TN>::LD;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) lds[acc_row(e, lane) * LD + 32 * j + (lane & 31)] = acc[j][e];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    constexpr int LANES = 8 * TN;                // lanes of a row, 4 columns each
    const int64_t col = col0 + 4 * (lane % LANES);
    const bool whole = vec && col + 4 <= g.n;
    f32x4 bias = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; q++)
        if (g.bias && col + q < g.n) bias[q] = g.bias[col + q];
#pragma unroll 2
    for (int r = lane / LANES; r < 32; r += 64 / LANES) {
        const int64_t row = row0 + r;
        if (row >= g.m) break;
        f32x4 z = *reinterpret_cast<const f32x4*>(lds + r * LD + 4 * (lane % LANES));
        const float t = (z[0] - z[0]) + (z[1] - z[1]) + (z[2] - z[2]) + (z[3] - z[3]);
        if (t != 0.f) {                          // NaN: some sum is not finite
            for (int q = 0; q < 4; q++) {
                const float v = lds[r * LD + 4 * (lane % LANES) + q];
                const float w = finite_f32(v) || col + q >= g.n ? v : plain_element<A_KC, B_KC>(g, row, col + q, 0, g.k);
                if (q == 0) z[0] = w; else if (q == 1) z[1] = w; else if (q == 2) z[2] = w; else z[3] = w;
            }
        }
        z += bias;
        f32x4 y;
#pragma unroll
        for (int q = 0; q < 4; q++) y[q] = act_value(g.act, z[q]);
        const f32x4 keep = saves_output(g.act) ? y : z;
        if (whole) {
            if (g.saved) *reinterpret_cast<f32x4*>(g.saved + row * g.lds + col) = keep;
            if (g.residual) y += *reinterpret_cast<const f32x4*>(g.residual + row * g.ldr + col);
            *reinterpret_cast<f32x4*>(g.c + row * g.ldc + col) = y;
        } else {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (col + q >= g.n) break;
                if (g.saved) g.saved[row * g.lds + col + q] = keep[q];
                if (g.residual) y[q] += g.residual[row * g.ldr + col + q];
                g.c[row * g.ldc + col + q] = y[q];
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
}

// ---------------------------------------------------------------------------------------------------- tiles through LDS
// One operand of R output rows, 16 of the contraction per stage.  LDS holds the three bf16 planes in fragment order: for each
// half of the 16 (kg) R x 16 bytes, so a fragment is one ds_read_b128 at consecutive addresses.
// KC: the contraction index is the fast one in memory (a thread takes 8 consecutive floats of one row, its neighbour the other
// half: the padding keeps the two halves' writes in different banks); otherwise the output index is (a thread takes 8 floats
// down one column).
template <bool KC, bool VEC, int R, int NT>
struct SplitOperand {
    static constexpr int KG = 16 * R + 64;
    static constexpr int PLANE = 2 * KG;
    static constexpr int BYTES = kPlanes * PLANE;
    static constexpr int PER = 2 * R / NT;                          // units (row, half of the 16) of a thread
    static_assert(2 * R % NT == 0, "whole units per thread");

    float reg[PER][8];
    // the next step's place: an address that is the same for the wavefront and an offset per unit that never changes
    const float* base[PER];
    unsigned off[PER];
    int64_t step;

    static __device__ __forceinline__ void unit(int tid, int i, int& row, int& kg) {
        const int u = tid + i * NT;
        if (KC) { row = u >> 1; kg = u & 1; } else { row = u % R; kg = __builtin_amdgcn_readfirstlane(u / R); }
    }
    // rows past the matrix are clamped: their products are not stored
    __device__ __forceinline__ void init(const float* __restrict__ p, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int tid) {
        step = KC ? 16 : 16 * ld;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            int row, kg;
            unit(tid, i, row, kg);
            const unsigned r = (unsigned)(min(row0 + row, rows - 1) - row0);
            base[i] = KC ? p + row0 * ld + k0 : p + (k0 + 8 * kg) * ld + row0;
            off[i] = KC ? 4u * (r * (unsigned)ld + 8u * kg) : 4u * r;
        }
    }
    static __device__ __forceinline__ const float* place(const float* b, unsigned o) {
        return reinterpret_cast<const float*>(reinterpret_cast<const char*>(b) + o);
    }
    // unit i of 16 of the contraction that are all there
    __device__ __forceinline__ void load(int i, int64_t ld) {
        if (KC && VEC) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(place(base[i], off[i])), y = *reinterpret_cast<const f32x4*>(place(base[i] + 4, off[i]));
#pragma unroll
            for (int e = 0; e < 4; e++) { reg[i][e] = x[e]; reg[i][4 + e] = y[e]; }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) reg[i][e] = *place(base[i] + (KC ? e : e * ld), off[i]);
        }
        base[i] += step;
    }
    // the last ones: `left` (1 to 15) are there, the others count as zero
    __device__ __forceinline__ void load_tail(int64_t ld, int left, int tid) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            int row, kg;
            unit(tid, i, row, kg);
#pragma unroll
            for (int e = 0; e < 8; e++) reg[i][e] = 8 * kg + e < left ? *place(base[i] + (KC ? e : e * ld), off[i]) : 0.f;
        }
    }
    // two of unit i's eight floats; with the last two the unit's pieces go to LDS
    __device__ __forceinline__ void split_part(int i, int part, u32x4 (&p)[kPlanes], char* lds, int tid) const {
        unsigned h, m, l;
        split_pair(reg[i][2 * part], reg[i][2 * part + 1], h, m, l);
        p[0][part] = h; p[1][part] = m; p[2][part] = l;
        if (part == 3) {
            int row, kg;
            unit(tid, i, row, kg);
#pragma unroll
            for (int q = 0; q < kPlanes; q++) *reinterpret_cast<u32x4*>(lds + q * PLANE + kg * KG + row * 16) = p[q];
        }
    }
    __device__ __forceinline__ void store(char* lds, int tid) const {
        u32x4 p[kPlanes];
#pragma unroll
        for (int i = 0; i < PER; i++)
#pragma unroll
            for (int part = 0; part < 4; part++) split_part(i, part, p, lds, tid);
    }
    // rows 32*b .. 32*b + 31
    static __device__ __forceinline__ void fragment(const char* lds, int b, int lane, u32x4 (&f)[kPlanes]) {
#pragma unroll
        for (int q = 0; q < kPlanes; q++)
            f[q] = *reinterpret_cast<const u32x4*>(lds + q * PLANE + (lane >> 5) * KG + (32 * b + (lane & 31)) * 16);
    }
};

template <int TM_, int TN_, int WM_, int WN_, int WGS_>
struct SplitTile {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, WGS = WGS_;   // WGS: wavefronts per SIMD the registers are held to
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, NT = 64 * WM * WN;
};
typedef SplitTile<2, 4, 4, 2, 2> Tile256;
typedef SplitTile<2, 2, 2, 2, 2> Tile128;

template <typename Cfg, bool A_KC, bool B_KC>
struct TileLds {
    static constexpr int STAGE = SplitOperand<A_KC, true, Cfg::BM, Cfg::NT>::BYTES + SplitOperand<B_KC, true, Cfg::BN, Cfg::NT>::BYTES;
    static constexpr int EPI = Cfg::WM * Cfg::WN * EpiBlock<Cfg::TN>::BYTES;
    static constexpr int BYTES = 2 * STAGE > EPI ? 2 * STAGE : EPI;
};

// Bound by the matrix cores, which are busy for 60 to 76 % of the cycles, at a clock that falls to 1.9 GHz: 8192 x 4096 over 1024
// with GELU and z kept 335 us (205 TFLOP/s; 268 MB of stores that little runs beside), its dX 307 us (224), its dW 319 us (215),
// 8192 x 1024 over 1024 with a residual 110 us (156; 49 % of the cycles).
// VEC: the operands whose contraction index is the fast one can be read 16 bytes at a time
template <typename Cfg, bool A_KC, bool B_KC, bool VEC>
__global__ __launch_bounds__(Cfg::NT, Cfg::WGS) void epilogue_tile_kernel(EpiArgs g, bool vec_c) {
    constexpr int TM = Cfg::TM, TN = Cfg::TN;
    using OpA = SplitOperand<A_KC, VEC, Cfg::BM, Cfg::NT>;
    using OpB = SplitOperand<B_KC, VEC, Cfg::BN, Cfg::NT>;
    constexpr int STAGE = TileLds<Cfg, A_KC, B_KC>::STAGE;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
    int tm, tn;
    tile_of(blockIdx.x, g.tiles_m, g.tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * Cfg::BM, n0 = (int64_t)tn * Cfg::BN;
    const int64_t kb = blockIdx.y * g.k_per_split, ke = min(g.k, kb + g.k_per_split);
    const int whole = ke > kb ? (int)((ke - kb) / 16) : 0, left = ke > kb ? (int)((ke - kb) % 16) : 0;
    const int steps = whole + (left ? 1 : 0);

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;

    OpA oa;
    OpB ob;
    oa.init(g.a, g.lda, m0, g.m, kb, tid);
    ob.init(g.b, g.ldb, n0, g.n, kb, tid);
    const auto fetch = [&](int s) {
        if (s < whole) {
#pragma unroll
            for (int i = 0; i < OpA::PER; i++) oa.load(i, g.lda);
#pragma unroll
            for (int i = 0; i < OpB::PER; i++) ob.load(i, g.ldb);
        } else if (s < steps) {
            oa.load_tail(g.lda, left, tid);
            ob.load_tail(g.ldb, left, tid);
        }
    };
    const auto put = [&](int s) {
        oa.store(smem + (s & 1) * STAGE, tid);
        ob.store(smem + (s & 1) * STAGE + OpA::BYTES, tid);
    };
    // A step's products, and between the 32 x 32 tiles' a share of the splitting of the next step's operands (in registers since
    // the step before) and of the loads of the one after: what a wavefront issues while the matrix core is busy costs nothing.
    const auto step = [&](int s, auto more) {
        const char* cur = smem + (s & 1) * STAGE;
        char* next = smem + (s & 1 ^ 1) * STAGE;
        u32x4 fa[2][kPlanes], fb[TN][kPlanes], planes[kPlanes];
        OpB::fragment(cur + OpA::BYTES, wn * TN, lane, fb[0]);
        OpA::fragment(cur, wm * TM, lane, fa[0]);
#pragma unroll
        for (int j = 1; j < TN; j++) OpB::fragment(cur + OpA::BYTES, wn * TN + j, lane, fb[j]);
        constexpr int PARTS = 4 * (OpA::PER + OpB::PER), TILES = TM * TN;
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            const int i = t / TN, j = t % TN;
            if (j == 0 && i + 1 < TM) OpA::fragment(cur, wm * TM + i + 1, lane, fa[(i + 1) & 1]);
            acc[i][j] = mfma_split(fa[i & 1], fb[j], acc[i][j]);
            if constexpr (decltype(more)::value) {
#pragma unroll
                for (int x = t * PARTS / TILES; x < (t + 1) * PARTS / TILES; x++) {
                    if (x < 4 * OpA::PER) {
                        oa.split_part(x / 4, x % 4, planes, next, tid);
                        if (x % 4 == 3) oa.load(x / 4, g.lda);
                    } else {
                        ob.split_part(x / 4 - OpA::PER, x % 4, planes, next + OpA::BYTES, tid);
                        if (x % 4 == 3) ob.load(x / 4 - OpA::PER, g.ldb);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __syncthreads();
    };
    if (steps > 0) {
        fetch(0);
        put(0);
        fetch(1);
    }
    __syncthreads();
    int s = 0;
    for (; s + 2 < whole; s++) step(s, std::true_type{});
    for (; s < steps; s++) {                     // the last two or three: what is left to load and to split
        if (s + 1 < steps) put(s + 1);
        fetch(s + 2);
        step(s, std::false_type{});
    }

    const int64_t row0 = m0 + wm * 32 * TM, col0 = n0 + wn * 32 * TN;
    if (g.splits > 1) {
        float* part = g.partial + (int64_t)blockIdx.y * g.m * g.n;
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int64_t row = row0 + 32 * i + acc_row(e, lane);
                if (row >= g.m) continue;
#pragma unroll
                for (int j = 0; j < TN; j++) {
                    const int64_t col = col0 + 32 * j + (lane & 31);
                    if (col < g.n) part[row * g.n + col] = acc[i][j][e];
                }
            }
        return;
    }
    float* block = reinterpret_cast<float*>(smem + wave * EpiBlock<TN>::BYTES);
#pragma unroll
    for (int i = 0; i < TM; i++) finish_block<TN, A_KC, B_KC>(g, acc[i], block, row0 + 32 * i, col0, lane, vec_c);
}

// the splits' partial sums, added in order, through the epilogue; bound by memory (8192 x 1024 in two parts 27 us)
template <bool A_KC, bool B_KC>
__global__ __launch_bounds__(256) void epilogue_fold_kernel(EpiArgs g) {
    const int64_t total = g.m * g.n;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float sum = 0.f;
        for (int s = 0; s < g.splits; s++) sum += g.partial[s * total + i];
        const int64_t row = i / g.n, col = i - row * g.n;
        if (!finite_f32(sum)) sum = plain_element<A_KC, B_KC>(g, row, col, 0, g.k);
        finish_element(g, row, col, sum);
    }
}

// ---------------------------------------------------------------------------------------------------- small products
// Outputs that fill few tiles: a workgroup owns a 32 x 32 tile and its wavefronts cut the contraction, each splitting its
// fragments straight from memory in registers; their sums meet in LDS.  No barrier and no LDS in the loop, so a wavefront
// keeps several steps' loads in flight, which is what such a product waits for: 1 x 4096 over 1024 (16.8 MB of weights) 7.6 us
// with the weights in the memory-side cache, 9.0 us without; 777 x 513 over 784 13.5 us.  (Loads a step further ahead, with the
// registers for it taken from the addresses, were slower: 14.5 us.)
template <bool KC>
__device__ __forceinline__ void direct_fragment(const float* __restrict__ p, int64_t ld, int64_t row, int64_t k, int64_t ke, bool vec,
                                                float (&x)[8]) {
    if (k + 8 <= ke) {
        if (KC) {
            const float* q = p + row * ld + k;
            if (vec) {
                const f32x4 u = *reinterpret_cast<const f32x4*>(q), v = *reinterpret_cast<const f32x4*>(q + 4);
#pragma unroll
                for (int e = 0; e < 4; e++) { x[e] = u[e]; x[4 + e] = v[e]; }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = q[e];
            }
        } else {
            const float* q = p + k * ld + row;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = q[e * ld];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = k + e < ke ? (KC ? p[row * ld + k + e] : p[(k + e) * ld + row]) : 0.f;
    }
}

template <int T_, int WAVES_>
struct SmallTile {
    static constexpr int T = T_, WAVES = WAVES_, SIZE = 32 * T, NT = 64 * WAVES;   // T x T blocks of 32 x 32
};
typedef SmallTile<1, 8> Small32;
typedef SmallTile<2, 8> Small64;
typedef SmallTile<1, 16> SmallLong;

template <typename Cfg, bool A_KC, bool B_KC>
__device__ __forceinline__ void small_tile(const EpiArgs& g, int tile, int split, bool vec_a, bool vec_b, float (&sums)[Cfg::WAVES][32 * 33]) {
    constexpr int T = Cfg::T, WAVES = Cfg::WAVES;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t m0 = (int64_t)(tile / g.tiles_n) * Cfg::SIZE, n0 = (int64_t)(tile % g.tiles_n) * Cfg::SIZE;
    const int64_t kb = split * g.k_per_split, ke = min(g.k, kb + g.k_per_split);
    int64_t row[T], col[T];                      // past the matrix the last one is read, its products are not stored
#pragma unroll
    for (int i = 0; i < T; i++) {
        row[i] = min(m0 + 32 * i + (lane & 31), g.m - 1);
        col[i] = min(n0 + 32 * i + (lane & 31), g.n - 1);
    }
    f32x16 acc[T][T];
#pragma unroll
    for (int i = 0; i < T; i++)
#pragma unroll
        for (int j = 0; j < T; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;
    // kDepth steps' loads are issued before the first one's products
    constexpr int kDepth = T == 1 && WAVES == 8 ? 2 : 1, kStep = 16 * WAVES;
    // a layer's bias gradient rides with its weight gradient: the first tile row's workgroups add up what they read of dz
    constexpr bool kSums = !A_KC && !B_KC;
    const bool wants = kSums && g.colsum && m0 == 0;
    float column[T];
#pragma unroll
    for (int i = 0; i < T; i++) column[i] = 0.f;
    const int64_t half = 8 * (lane >> 5);
    for (int64_t k = kb + 16 * wave; k < ke; k += kDepth * kStep) {
        float x[kDepth][T][8], y[kDepth][T][8];
#pragma unroll
        for (int d = 0; d < kDepth; d++)
#pragma unroll
            for (int i = 0; i < T; i++) {
                direct_fragment<A_KC>(g.a, g.lda, row[i], k + d * kStep + half, ke, vec_a, x[d][i]);
                direct_fragment<B_KC>(g.b, g.ldb, col[i], k + d * kStep + half, ke, vec_b, y[d][i]);
            }
#pragma unroll
        for (int d = 0; d < kDepth; d++) {
            if constexpr (kSums)
                if (wants) {
#pragma unroll
                    for (int i = 0; i < T; i++)
                        column[i] += ((y[d][i][0] + y[d][i][1]) + (y[d][i][2] + y[d][i][3])) + ((y[d][i][4] + y[d][i][5]) + (y[d][i][6] + y[d][i][7]));
                }
            u32x4 fa[T][kPlanes], fb[T][kPlanes];
#pragma unroll
            for (int i = 0; i < T; i++) { split_eight(x[d][i], fa[i]); split_eight(y[d][i], fb[i]); }
#pragma unroll
            for (int i = 0; i < T; i++)
#pragma unroll
                for (int j = 0; j < T; j++) acc[i][j] = mfma_split(fa[i], fb[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < T; i++)
#pragma unroll
        for (int j = 0; j < T; j++) {
            if (i + j > 0) __syncthreads();
#pragma unroll
            for (int e = 0; e < 16; e++) sums[wave][acc_row(e, lane) * 33 + (lane & 31)] = acc[i][j][e];
            __syncthreads();
            for (int q = tid; q < 32 * 32; q += Cfg::NT) {
                const int64_t r = m0 + 32 * i + (q >> 5), c = n0 + 32 * j + (q & 31);
                if (r >= g.m || c >= g.n) continue;
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < WAVES; w++) s += sums[w][(q >> 5) * 33 + (q & 31)];
                if (g.splits > 1) {
                    g.partial[((int64_t)split * g.m + r) * g.n + c] = s;
                } else {
                    if (!finite_f32(s)) s = plain_element<A_KC, B_KC>(g, r, c, 0, g.k);
                    finish_element(g, r, c, s);
                }
            }
        }
    if constexpr (kSums)
        if (wants) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < T; i++) {
                const float both = column[i] + __shfl_xor(column[i], 32, 64);
                if (lane < 32) sums[wave][32 * i + lane] = both;
            }
            __syncthreads();
            if (tid < 32 * T && n0 + tid < g.n) {
                float t = 0.f;
#pragma unroll
                for (int w = 0; w < WAVES; w++) t += sums[w][tid];
                g.colsum[n0 + tid] = g.colsum_add ? g.colsum[n0 + tid] + t : t;
            }
        }
}

template <typename Cfg, bool A_KC, bool B_KC>
__global__ __launch_bounds__(Cfg::NT) void epilogue_small_kernel(EpiArgs g, bool vec_a, bool vec_b) {
    __shared__ float sums[Cfg::WAVES][32 * 33];
    small_tile<Cfg, A_KC, B_KC>(g, blockIdx.x, blockIdx.y, vec_a, vec_b, sums);
}

// A layer's two gradients in one launch, where each alone leaves compute units idle: dx (first workgroups) and dW
__global__ __launch_bounds__(SmallLong::NT) void epilogue_pair_kernel(EpiArgs dx, EpiArgs dw, bool vec_z, bool vec_w) {
    __shared__ float sums[SmallLong::WAVES][32 * 33];
    const int first = dx.tiles_m * dx.tiles_n, id = blockIdx.x;
    if (id < first) small_tile<SmallLong, true, true>(dx, id, 0, vec_z, vec_w, sums);
    else small_tile<SmallLong, false, false>(dw, id - first, 0, false, false, sums);
}

// ---------------------------------------------------------------------------------------------------- choice and launch
static int g_force_variant = -1, g_force_splits = 0, g_force_pair = -1;
constexpr int64_t kMostTiles = (1 << 22) - 1;             // of one launch: at 1024 threads each the threads are counted in 32 bits

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename Cfg, bool A_KC, bool B_KC, bool VEC>
static int launch_tile(const EpiArgs& g, bool vc) {
    constexpr int bytes = TileLds<Cfg, A_KC, B_KC>::BYTES;
    static bool raised = false;                 // more than 64 KB of LDS has to be asked for once
    if (!raised) {
        const int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(&epilogue_tile_kernel<Cfg, A_KC, B_KC, VEC>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "bh_gemm_epilogue: LDS size");
        if (rc) return rc;
        raised = true;
    }
    hipLaunchKernelGGL((epilogue_tile_kernel<Cfg, A_KC, B_KC, VEC>), dim3((unsigned)(g.tiles_m * g.tiles_n), (unsigned)g.splits), dim3(Cfg::NT),
                       bytes, stream(), g, vc);
    return BH_LAUNCH_CHECK("bh_gemm_epilogue");
}
template <typename Cfg, bool A_KC, bool B_KC>
static int launch_tile(const EpiArgs& g, bool va, bool vb, bool vc) {
    if constexpr (A_KC || B_KC)
        if ((A_KC && !va) || (B_KC && !vb)) return launch_tile<Cfg, A_KC, B_KC, false>(g, vc);
    return launch_tile<Cfg, A_KC, B_KC, true>(g, vc);
}

enum { kTile256 = 0, kTile128, kSmall32, kSmall64, kSmallLong, kVariants };
struct TileSize { int m, n; };
static const TileSize kSizes[kVariants] = {{Tile256::BM, Tile256::BN}, {Tile128::BM, Tile128::BN}, {32, 32}, {64, 64}, {32, 32}};

template <typename Cfg, bool A_KC, bool B_KC>
static int launch_small(const EpiArgs& g, bool va, bool vb) {
    hipLaunchKernelGGL((epilogue_small_kernel<Cfg, A_KC, B_KC>), dim3((unsigned)(g.tiles_m * g.tiles_n), (unsigned)g.splits), dim3(Cfg::NT), 0,
                       stream(), g, va, vb);
    return BH_LAUNCH_CHECK("bh_gemm_epilogue");
}

template <bool A_KC, bool B_KC>
static int run_product(EpiArgs g, int variant, int splits) {
    const bool va = A_KC && g.lda % 4 == 0 && aligned16(g.a), vb = B_KC && g.ldb % 4 == 0 && aligned16(g.b);
    const bool vc = g.ldc % 4 == 0 && aligned16(g.c) && (!g.saved || (g.lds % 4 == 0 && aligned16(g.saved))) &&
                    (!g.residual || (g.ldr % 4 == 0 && aligned16(g.residual)));
    const int64_t tiles_m = ceil_div(g.m, kSizes[variant].m), tiles_n = ceil_div(g.n, kSizes[variant].n);
    if (tiles_m * tiles_n > kMostTiles) return set_error(BH_EINVAL, "bh_gemm_epilogue: output too large");
    g.tiles_m = (int)tiles_m;
    g.tiles_n = (int)tiles_n;
    g.k_per_split = ceil_div(ceil_div(g.k > 0 ? g.k : 1, splits), 16) * 16;
    g.splits = (int)ceil_div(g.k > 0 ? g.k : 1, g.k_per_split);
    Scratch part;
    if (g.splits > 1) {
        if (!part.get(sizeof(float) * (size_t)g.splits * (size_t)(g.m * g.n))) return BH_ENOMEM;
        g.partial = (float*)part.p;
    }
    int rc;
    if (variant == kTile256) rc = launch_tile<Tile256, A_KC, B_KC>(g, va, vb, vc);
    else if (variant == kTile128) rc = launch_tile<Tile128, A_KC, B_KC>(g, va, vb, vc);
    else if (variant == kSmall64) rc = launch_small<Small64, A_KC, B_KC>(g, va, vb);
    else if (variant == kSmallLong) rc = launch_small<SmallLong, A_KC, B_KC>(g, va, vb);
    else rc = launch_small<Small32, A_KC, B_KC>(g, va, vb);
    if (rc || g.splits == 1) return rc;
    const int64_t blocks = ceil_div(g.m * g.n, 256);
    hipLaunchKernelGGL((epilogue_fold_kernel<A_KC, B_KC>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, stream(), g);
    return BH_LAUNCH_CHECK("bh_gemm_epilogue: fold");
}

// What a variant is expected to take, in us, so that the fastest is chosen.  A workgroup's steps (16 of the contraction; a small
// tile's wavefronts take that many each) last `alone` where it has the compute unit to itself, and `shared` times the workgroups
// on the unit where they fill it; each output tile costs `finish`, the launch `fixed`, and an operand that is read along its
// rows makes the steps `rows` longer.  A cut contraction adds a launch and its partial sums' traffic.  Fitted to 520 shapes of
// 1 to 8192 rows and 60 to 4100 features, all variants and cuts, three layouts: the choice is 2 % over the best one in the
// mean, 8 % at most for nine shapes in ten.
struct Cost { float alone, shared, finish, fixed, rows; int per_cu, waves; };
static const Cost kCost[kVariants] = {
    {2.05f, 2.05f, 9.65f, 4.67f, 0.f, 1, 1},       // 256 x 256
    {0.74f, 0.641f, 1.58f, 7.85f, 0.f, 3, 1},      // 128 x 128
    {0.015f, 0.609f, 1.11f, 2.20f, 0.232f, 2, 8},  // 32 x 32
    {1.76f, 1.37f, 4.17f, 0.56f, 0.073f, 1, 8},    // 64 x 64, wavefronts cut the contraction
    {1.19f, 0.501f, 1.12f, 1.11f, 0.125f, 1, 16},  // 32 x 32, twice the wavefronts
};
static double cost_of(int variant, int64_t m, int64_t n, int64_t k, int splits, int along_rows) {
    const Cost& c = kCost[variant];
    const int64_t per_split = ceil_div(ceil_div(k, splits), 16) * 16;
    const double cuts = (double)ceil_div(k, per_split);
    const double wgs = (double)ceil_div(m, kSizes[variant].m) * (double)ceil_div(n, kSizes[variant].n) * cuts;
    const double steps = (double)ceil_div(per_split, 16 * c.waves), slow = 1.0 + c.rows * along_rows;
    const double full = floor(wgs / (256.0 * c.per_cu)), rest = ceil((wgs - full * 256.0 * c.per_cu) / 256.0);
    double t = c.fixed;
    if (full > 0) t += full * (steps * slow * fmax(c.alone, c.per_cu * c.shared) + c.per_cu * c.finish);
    if (rest > 0) t += steps * slow * fmax(c.alone, rest * c.shared) + rest * c.finish;
    if (cuts > 1) t += 3.2 + 1.07e-6 * cuts * (double)m * (double)n;
    return t;
}
static double choose(int64_t m, int64_t n, int64_t k, int along_rows, int& variant, int& splits) {
    static const int kCuts[] = {1, 2, 3, 4, 6, 8, 12, 16, 32};
    double best = 1e30;
    variant = kTile256;
    splits = 1;
    for (int v = 0; v < kVariants; v++) {
        const double flops = 2.0 * (double)m * (double)n * (double)k;
        if ((v == kSmallLong && k < 256) || ((v == kSmall32 || v == kSmallLong) && flops > 2e10) || (v == kSmall64 && flops > 1e11)) continue;
        const int64_t tiles = ceil_div(m, kSizes[v].m) * ceil_div(n, kSizes[v].n);
        if (tiles > kMostTiles) continue;
        for (int s : kCuts) {
            if (s > 1 && (k / s < 64 || tiles * s > 2048 || (double)s * m * n > 1.3e8)) break;
            const double t = cost_of(v, m, n, k > 0 ? k : 1, s, along_rows);
            if (t < best) { best = t; variant = v; splits = s; }
        }
    }
    return best;
}

static void pick(int trans_a, int trans_b, const EpiArgs& g, int& variant, int& splits) {
    constexpr int64_t kMaxLd = (int64_t)1 << 22;   // 256 rows of a tile within 32 bits of bytes; past it the small tiles' addresses
    choose(g.m, g.n, g.k, (trans_a ? 1 : 0) + (trans_b ? 0 : 1), variant, splits);
    if (g_force_variant >= 0) { variant = g_force_variant; splits = 1; }
    if (g_force_splits > 0) splits = g_force_splits;
    if (variant <= kTile128 && (g.lda >= kMaxLd || g.ldb >= kMaxLd)) { variant = kSmall64; splits = 1; }
}
static int product(int trans_a, int trans_b, const EpiArgs& g, int variant, int splits) {
    if (!trans_a) return trans_b ? run_product<true, true>(g, variant, splits) : run_product<true, false>(g, variant, splits);
    return trans_b ? run_product<false, true>(g, variant, splits) : run_product<false, false>(g, variant, splits);
}

// dx[m,k] and dw[k,n] in one launch
static int launch_pair(EpiArgs dx, EpiArgs dw, bool vz, bool vw) {
    for (EpiArgs* g : {&dx, &dw}) {
        g->tiles_m = (int)ceil_div(g->m, SmallLong::SIZE);
        g->tiles_n = (int)ceil_div(g->n, SmallLong::SIZE);
        g->k_per_split = g->k;
        g->splits = 1;
    }
    const int tiles = dx.tiles_m * dx.tiles_n + dw.tiles_m * dw.tiles_n;
    hipLaunchKernelGGL(epilogue_pair_kernel, dim3((unsigned)tiles), dim3(SmallLong::NT), 0, stream(), dx, dw, vz, vw);
    return BH_LAUNCH_CHECK("bh_dense_act_backward");
}
// Is one launch of sixteen-wavefront tiles expected to be faster than a launch for each gradient?  In the terms of cost_of, steps
// at three times the price (tiles of two products share less), against the two choices' sum.  Over 70 shapes of 1 to 8192 rows and
// 60 to 4100 features the time is 0.82 of two launches' in the mean (0.81 where the faster is always taken): us, one / two
// launches, 128 x 512 x 512 7 / 12, 32 x 784 x 128 7 / 9, 1000 x 300 x 300 12 / 15, 777 x 784 x 513 32 / 29, 512 x 1024 x 1024 39 / 32.
static bool in_one_launch(int64_t m, int64_t k, int64_t n) {
    const double tx = (double)ceil_div(m, 32) * (double)ceil_div(k, 32), tw = (double)ceil_div(k, 32) * (double)ceil_div(n, 32);
    if (tx + tw > (double)kMostTiles) return false;
    if (g_force_pair >= 0) return g_force_pair == 1;
    int variant, splits;
    const double two = choose(m, k, n, 0, variant, splits) + choose(k, n, m, 2, variant, splits);
    const Cost& c = kCost[kSmallLong];
    const double sx = (double)ceil_div(n, 16 * c.waves), sw = (double)ceil_div(m, 16 * c.waves) * (1 + 2 * c.rows);
    const double work = (tx * (3 * sx * c.shared + c.finish) + tw * (3 * sw * c.shared + c.finish)) / 256;
    const double tail = tx + tw > 256 ? 0.5 * (fmin(sx, sw) * c.shared + c.finish) : 0;
    return c.fixed + 1.5 + fmax(fmax(sx, sw) * c.alone + c.finish, work + tail) < two + 2;
}

}  // namespace bh

using namespace bh;

extern "C" {

int bh_gemm_epilogue(int trans_a, int trans_b, int64_t m, int64_t n, int64_t k, const float* a, int64_t lda, const float* b, int64_t ldb,
                     float* c, int64_t ldc, const float* bias, int act, float* saved, int64_t lds, const float* residual, int64_t ldr) {
    BH_CHECK_ARG(m >= 0 && n >= 0 && k >= 0, "negative dimension");
    BH_CHECK_ARG(act >= BH_ACT_NONE && act <= BH_ACT_GELU, "unknown activation");
    if (m == 0 || n == 0) return BH_OK;
    BH_CHECK_ARG(c && ((a && b) || k == 0), "null pointer");
    BH_CHECK_ARG(lda >= (trans_a ? m : k) && ldb >= (trans_b ? k : n) && ldc >= n, "leading dimension too small");
    BH_CHECK_ARG((!saved || lds >= n) && (!residual || ldr >= n), "leading dimension too small");
    BH_CHECK_ARG(residual != c || ldr == ldc, "a residual in place has the output's leading dimension");
    BH_REQUIRE_INIT();
    BH_CALL_GUARD();
    ProfScope prof(BH_PROF_GEMM, 2.0 * (double)m * (double)n * (double)k);
    EpiArgs g = {};
    g.a = a; g.b = b; g.m = m; g.n = n; g.k = k; g.lda = lda; g.ldb = ldb; g.c = c; g.ldc = ldc; g.bias = bias;
    g.saved = saved; g.lds = lds; g.residual = residual; g.ldr = ldr; g.act = act;
    int variant, splits;
    pick(trans_a, trans_b, g, variant, splits);
    return product(trans_a, trans_b, g, variant, splits);
}

int bh_dense_act_backward(int act, const float* x, const float* w, const float* saved, const float* dy, float* dx, float* gw, float* gb,
                          int64_t m, int64_t k, int64_t n, int accumulate) {
    BH_CHECK_ARG(m >= 0 && k >= 0 && n >= 0, "negative dimension");
    BH_CHECK_ARG(act >= BH_ACT_NONE && act <= BH_ACT_GELU, "unknown activation");
    BH_CHECK_ARG((dy && (!dx || w) && (!gw || x) && (act == BH_ACT_NONE || saved)) || m == 0 || n == 0, "null pointer");
    BH_REQUIRE_INIT();
    BH_CALL_GUARD();
    EpiArgs a = {}, b = {};                                   // dx[m,k] = dz[m,n] . w[k,n]^T,  gw[k,n] (+)= x[m,k]^T . dz[m,n]
    a.b = w; a.lda = n; a.ldb = n; a.c = dx; a.ldc = k; a.m = m; a.n = k; a.k = n; a.act = BH_ACT_NONE;
    b.a = x; b.lda = k; b.ldb = n; b.c = gw; b.ldc = n; b.m = k; b.n = n; b.k = m; b.act = BH_ACT_NONE;
    b.residual = accumulate ? gw : nullptr; b.ldr = n;
    const bool whole = m > 0 && k > 0 && n > 0, one = whole && (dx || gw) && in_one_launch(m, k, n);
    int variant = kSmallLong, splits = 1;
    if (gw && whole && !one) pick(1, 0, b, variant, splits);
    // db = the column sums of dz: with dW where small tiles make that whole, else with dz (or alone)
    const bool rides = gb && gw && whole && variant >= kSmall32 && splits == 1;
    if (rides) { b.colsum = gb; b.colsum_add = accumulate ? 1 : 0; }
    // dz = dy * act'(z)
    const float* dz = dy;
    Scratch own;
    int rc = BH_OK;
    if (act != BH_ACT_NONE && m > 0 && n > 0 && (dx || gw || gb)) {
        if (!own.get(sizeof(float) * (size_t)(m * n))) return BH_ENOMEM;
        rc = gb && !rides ? bh_activation_backward_colsum(act, saved, dy, (float*)own.p, gb, m, n, accumulate)
                          : bh_activation_backward(act, saved, dy, (float*)own.p, m * n, 0);
        dz = (const float*)own.p;
    } else if (gb && n > 0 && !rides) {
        rc = m > 0 ? bh_colsum(dy, gb, m, n, accumulate) : accumulate ? BH_OK : bh_fill(gb, 0.f, n);
    }
    if (rc != BH_OK) return rc;
    a.a = dz;
    b.b = dz;
    if (one) {
        // also for one of the two: its bits do not depend on whether the other is asked for
        ProfScope prof(BH_PROF_GEMM, (dx && gw ? 4.0 : 2.0) * (double)m * (double)n * (double)k);
        if (!dx) a.m = 0;
        if (!gw) b.m = 0;
        return launch_pair(a, b, n % 4 == 0 && aligned16(dz), n % 4 == 0 && aligned16(w));
    }
    // n == 0: zeros
    if (dx) rc = bh_gemm_epilogue(0, 1, m, k, n, dz, n, w, n, dx, k, nullptr, BH_ACT_NONE, nullptr, 0, nullptr, 0);
    if (rc != BH_OK || !gw) return rc;
    // m == 0: zeros
    if (!whole) return bh_gemm_epilogue(1, 0, k, n, m, x, k, dz, n, gw, n, nullptr, BH_ACT_NONE, nullptr, 0, accumulate ? gw : nullptr, n);
    ProfScope prof(BH_PROF_GEMM, 2.0 * (double)m * (double)n * (double)k);
    return product(1, 0, b, variant, splits);
}

int bh_gemm_epilogue_force(int variant, int splits) {
    BH_CHECK_ARG(variant >= -1 && variant < kVariants && splits >= 0 && splits <= 64, "variant -1 to 4, 0 to 64 splits");
    g_force_variant = variant;
    g_force_splits = splits;
    return BH_OK;
}

int bh_dense_act_backward_force(int pair) {
    BH_CHECK_ARG(pair >= -1 && pair <= 1, "-1, 0 or 1");
    g_force_pair = pair;
    return BH_OK;
}

}  // extern "C"
