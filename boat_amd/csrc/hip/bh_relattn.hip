// bh_relattn.hip - attention with a learned relative position bias by buckets, forward and backward.
//
// For query i, key j of head h:  x = scale q_i.k_j + T[bucket(j - (i + offset))][h],  P = softmax over the keys a query may see,
// O = P V.  Backward from the rows' log-sum-exp (as bh_sdpa_backward: P = exp(x - lse), nothing of size [sq, sk] is stored):
//   dV = P^T dO,  dP = dO V^T,  dS = P o (dP - rowsum(dO o O)),  dQ = scale dS K,  dK = scale dS^T Q,
//   dT[b][h] = sum of dS over the batch and all (i, j) whose relative position falls into bucket b.
// The bias has the value of one table entry along every diagonal and is constant beyond the last border, so it is never
// stored either: a wavefront's 32 x 32 block of scores has 63 diagonals, whose values 63 lanes look up; blocks past the last
// border (all but a band around the diagonal) add one number.  Its gradient is the blocks' diagonal sums, in the same way.
//
// All products run on the bf16 matrix cores from operands split into three bf16 each (bh_split.h).  Scores are computed
// with the operand that varies along the second product's contraction as the rows, so that a lane's accumulators are
// already, after the exponential, its fragment of the next product: the contraction index of that product is dealt out in the
// accumulators' order (rows 16 s + 4 half + 0..3 and 16 s + 8 + 4 half + 0..3), and the other operand is staged in the same.
//
// Every key and value is used by all the query tiles of its head (and every query by all key tiles in the backward pass), so
// the split is made once: a first kernel writes the operands' planes to work memory in the order in which fragments are read
// (padded with zeros to whole blocks, so strides, odd sizes and padding end there), and the tile kernels move blocks of it
// straight into LDS, without a register or an arithmetic instruction.  A few query rows over a long history would read more
// that way than the history itself: they take a kernel that splits in registers what each wavefront reads once.
#include "bh_split.h"

#include <math.h>

namespace bh {

constexpr int kMaxBuckets = 256;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kMaskedBias = -1e30f;      // a table value this low masks its bucket, like -inf

// the buckets' borders: distance n < exact is its own bucket; from there bucket exact + j starts at border[j]
struct Buckets {
    int exact, far, side, last;            // far: logarithmic buckets; side: buckets of one direction; last = border[far - 1]
    int both;
    int line;                              // relative positions from the last border (and a block) on one side to the other's, or 0
    float log2_exact, per_log2;
    int border[kMaxBuckets / 2 + 1];
};

struct RelArgs {
    const float *q, *k, *v, *table, *out_in, *lse_in, *d_out;
    const int32_t* kv_len;
    float *out, *lse, *dq, *dk, *dv;
    int64_t qs[3], ks[3], vs[3], os[3];    // strides of batch, head, row
    int batch, heads, kv_heads, group, d;
    int64_t sq, sk, offset;
    int at_end;                            // the offset counts from a sequence's own last sq keys
    int causal;
    float scale;
    bool vec_q, vec_k, vec_v, vec_o;
    int splits; int64_t keys_per_split;    // few workgroups (forward, dQ): partial results per split of the keys
    float *part_o, *part_ml;               // [split][batch*heads*sq][d], [split][batch*heads*sq][2]
    float* delta;                          // backward: rowsum(dO o O)
    double* part_table;                    // backward: [split][batch*heads][query tiles][buckets]
    int buckets, q_tiles;
    const char *k_row, *k_col, *v_row, *v_col, *q_row, *q_col, *g_row, *g_col;   // planes
    int k_blocks, q_blocks;                // of 32 rows, per head
    float* part_q;                         // backward over split keys: [split][batch*heads][sq][d]
    int q_splits, queries_per_split;       // dK, dV: splits of the queries
    float *part_k, *part_v;                // shared key heads or split queries: [split][batch*heads][sk][d]
    Buckets b;
};

// valid keys of a sequence, and the position of its first query
__device__ __forceinline__ int length_of(const RelArgs& g, int bt) {
    return g.kv_len ? __builtin_amdgcn_readfirstlane(min(max(g.kv_len[bt], 0), (int)g.sk)) : (int)g.sk;
}
__device__ __forceinline__ int64_t offset_of(const RelArgs& g, int len) { return g.at_end ? g.offset + len - g.sq : g.offset; }

// ---- the bias as a workgroup sees it.  Where the borders span no more than kLine relative positions LDS holds the bias (times
// log2 e) and the bucket of each of them, worked out once; else the borders and the head's table column, and every wavefront
// looks its blocks' diagonals up.  With a line / with lookups, 32 buckets to distance 128, us: 128 heads of 1024 forward 203 / 205,
// causal with backward 586 / 593; 5 KB of LDS let two workgroups share a compute unit at every head size.
constexpr int kLine = 1024;

__device__ __forceinline__ int bucket_of(const Buckets& b, const int* border, int rel) {
    const int n = b.both ? abs(rel) : max(-rel, 0);
    int f = (int)((__builtin_amdgcn_logf((float)max(n, 1)) - b.log2_exact) * b.per_log2);   // right up to one, the borders decide
    f = min(max(f, 0), b.far - 1);
    if (n < border[f]) f--;
    else if (n >= border[f + 1]) f++;      // border[far] is past every distance
    const int one = n < b.exact ? n : b.exact + f;
    return b.both && rel > 0 ? b.side + one : one;
}
__device__ __forceinline__ float table_value(const RelArgs& g, int bucket, int head) {
    const float t = g.table[(int64_t)bucket * g.heads + head];
    return t <= kMaskedBias ? -INFINITY : t * kLog2e;
}
// does every relative position of [lo, hi] fall into one bucket?  Which one, or -1
__device__ __forceinline__ int constant_bucket(const Buckets& b, int64_t lo, int64_t hi) {
    if (hi <= -(int64_t)b.last) return b.side - 1;
    if (b.both) return lo >= b.last ? 2 * b.side - 1 : -1;
    return lo >= 0 ? 0 : -1;
}
struct Bias {
    static constexpr int WINDOW = 4 * (kMaxBuckets / 2 + 4) + 4 * kMaxBuckets;   // borders and column, then 64 floats a wavefront
    static constexpr int BYTES = 5 * kLine;
    static_assert(WINDOW + 4 * 64 * 4 <= BYTES, "four wavefronts");

    char* lds;
    int first;                             // relative position of the line's start
    float before, behind;                  // past the last border: keys before the query, keys behind it
    bool line;

    // to be followed by a barrier
    __device__ __forceinline__ Bias(const RelArgs& g, int head, char* area, int threads)
        : lds(area), first(-(g.b.last + 63)), before(table_value(g, g.b.side - 1, head)),
          behind(table_value(g, g.b.both ? 2 * g.b.side - 1 : 0, head)), line(g.b.line > 0) {
        if (line) {
            for (int i = threadIdx.x; i < g.b.line; i += threads) {
                const int k = bucket_of(g.b, g.b.border, first + i);
                reinterpret_cast<float*>(lds)[i] = table_value(g, k, head);
                reinterpret_cast<unsigned char*>(lds)[4 * kLine + i] = (unsigned char)k;
            }
        } else {
            int* border = reinterpret_cast<int*>(lds);
            float* value = reinterpret_cast<float*>(lds + 4 * (kMaxBuckets / 2 + 4));
            for (int i = threadIdx.x; i <= g.b.far; i += threads) border[i] = g.b.border[i];
            for (int i = threadIdx.x; i < g.buckets; i += threads) value[i] = table_value(g, i, head);
        }
    }
    __device__ __forceinline__ int bucket(const Buckets& b, int rel) const {
        return line ? reinterpret_cast<const unsigned char*>(lds)[4 * kLine + rel - first] : bucket_of(b, reinterpret_cast<const int*>(lds), rel);
    }
    // the biases of relative positions rel0 - 31 .. rel0 + 31 (a block that is not constant), for one wavefront
    __device__ __forceinline__ const float* diagonals(const Buckets& b, int rel0, int wave, int lane) const {
        if (line) return reinterpret_cast<const float*>(lds) + (rel0 - 31 - first);
        const float* value = reinterpret_cast<const float*>(lds + 4 * (kMaxBuckets / 2 + 4));
        float* win = reinterpret_cast<float*>(lds + WINDOW) + 64 * wave;
        const float t = value[bucket_of(b, reinterpret_cast<const int*>(lds), rel0 + lane - 31)];
        __builtin_amdgcn_wave_barrier();
        win[lane] = t;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        return win;
    }
};

// ---- loading.  Eight floats of a row from element c on; places past d, and rows that are not `live`, are zero
__device__ __forceinline__ void row_eight(const float* __restrict__ p, bool live, int c, int d, bool vec, float (&x)[8]) {
    if (live && vec && c + 8 <= d) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p + c), b = *reinterpret_cast<const f32x4*>(p + c + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) { x[e] = a[e]; x[4 + e] = b[e]; }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = live && c + e < d ? p[c + e] : 0.f;
    }
}
// ---- planes in work memory.  Per 32 rows of an operand (zero past its rows and past d), 192 * DP bytes each:
//   row form     [plane][chunk of 8 of d][row]           16-byte pieces: fragments whose contraction runs along d
//   column form  [plane][step of 16 rows][half][of d]    16-byte pieces: fragments whose contraction runs over the rows
template <int DP> struct Block {
    static constexpr int PLANE = 64 * DP;                // bytes of 32 rows
    static constexpr int BYTES = kPlanes * PLANE;
    static __device__ __forceinline__ void row_fragment(const char* p, int s, int lane, u32x4 (&f)[kPlanes]) {
#pragma unroll
        for (int q = 0; q < kPlanes; q++)
            f[q] = *reinterpret_cast<const u32x4*>(p + q * PLANE + (2 * s + (lane >> 5)) * 512 + (lane & 31) * 16);
    }
    // rows (of d) 32*b + 0..31, contraction step s
    static __device__ __forceinline__ void column_fragment(const char* p, int b, int s, int lane, u32x4 (&f)[kPlanes]) {
#pragma unroll
        for (int q = 0; q < kPlanes; q++)
            f[q] = *reinterpret_cast<const u32x4*>(p + q * PLANE + ((2 * s + (lane >> 5)) * DP + 32 * b + (lane & 31)) * 16);
    }
};

struct SplitJob {
    const float* src; int64_t s[3];                      // strides of batch, head, row
    int heads; int64_t rows;
    const int32_t* len;                                  // valid rows per batch entry, or NULL
    int blocks;                                          // of 32 rows, per head
    char* row; char* col;                                // either may be NULL
    bool vec;
    const float* with; float* dots;                      // dots [head][row] = the row's product with the same row of `with`, or NULL
};
constexpr int kMaxJobs = 4;
struct SplitJobs { SplitJob j[kMaxJobs]; int first[kMaxJobs + 1]; int d; };   // first: workgroup number at which a job starts

// one block of 32 rows a workgroup: read once, written in the forms asked for.  Bound by memory: keys and values of 128 heads of
// 1024 at head size 64 (168 MB read and written) 27 us, all four operands of the backward pass (520 MB) 55 us.
template <int DP>
__global__ __launch_bounds__(256) void relattn_split_kernel(SplitJobs a) {
    __shared__ float x[32][DP + 4];
    int n = 0;
    while (n + 1 < kMaxJobs && (int)blockIdx.x >= a.first[n + 1]) n++;
    const SplitJob& j = a.j[n];
    const int id = blockIdx.x - a.first[n], bh = id / j.blocks, blk = id % j.blocks, bt = bh / j.heads, h = bh % j.heads;
    const int64_t rows = j.len ? min((int64_t)max(j.len[bt], 0), j.rows) : j.rows;
    const int64_t row0 = 32 * (int64_t)blk;
    if (j.len && row0 >= (rows + 63) / 64 * 64) return;  // never read
    const float* src = j.src + bt * j.s[0] + h * j.s[1] + row0 * j.s[2];
    const int live = (int)max((int64_t)0, min(rows - row0, (int64_t)32));
    for (int i = threadIdx.x; i < 32 * (DP / 4); i += 256) {
        const int r = i / (DP / 4), c = 4 * (i % (DP / 4));
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (r < live) {
            if (j.vec) {
                if (c < a.d) v = *reinterpret_cast<const f32x4*>(src + r * j.s[2] + c);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (c + e < a.d) v[e] = src[r * j.s[2] + c + e];
            }
        }
        *reinterpret_cast<f32x4*>(&x[r][c]) = v;
    }
    __syncthreads();
    if (j.dots) {                                        // eight lanes a row
        const int r = threadIdx.x >> 3;
        float t = 0.f;
        if (r < live) {
            const float* w = j.with + bt * j.s[0] + h * j.s[1] + (row0 + r) * j.s[2];
            for (int c = threadIdx.x & 7; c < a.d; c += 8) t += x[r][c] * w[c];
        }
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) t += __shfl_xor(t, off, 64);
        if (r < live && (threadIdx.x & 7) == 0) j.dots[(int64_t)bh * j.rows + row0 + r] = t;
    }
    const int64_t at = ((int64_t)bh * j.blocks + blk) * Block<DP>::BYTES;
    if (j.row)
        for (int i = threadIdx.x; i < 32 * (DP / 8); i += 256) {
            const int r = i & 31, c = i >> 5;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = x[r][8 * c + e];
            u32x4 p[kPlanes];
            split_eight<true>(y, p);
#pragma unroll
            for (int q = 0; q < kPlanes; q++) *reinterpret_cast<u32x4*>(j.row + at + q * Block<DP>::PLANE + i * 16) = p[q];
        }
    if (j.col)
        for (int i = threadIdx.x; i < 4 * DP; i += 256) {
            const int c = i % DP, sh = i / DP, r0 = 16 * (sh >> 1) + 4 * (sh & 1);
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = x[r0 + (e < 4 ? e : e + 4)][c];
            u32x4 p[kPlanes];
            split_eight<true>(y, p);
#pragma unroll
            for (int q = 0; q < kPlanes; q++) *reinterpret_cast<u32x4*>(j.col + at + q * Block<DP>::PLANE + i * 16) = p[q];
        }
}

// ---- work memory straight into LDS: a wavefront's instruction moves 1 KB, 16 bytes a lane, to consecutive LDS addresses
typedef __attribute__((address_space(3))) void* lds_ptr_t;
template <int KB, int WAVES>
__device__ __forceinline__ void copy_to_lds(const char* src, const char* lds, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < (KB + WAVES - 1) / WAVES; i++) {
        const int n = wave + i * WAVES;
        if (KB % WAVES != 0 && n >= KB) break;
        // M0 carries the LDS address; it is reserved, the compiler keeps nothing of its own in it in these kernels
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                     ::"v"(16u * (unsigned)lane), "s"(src + 1024 * n),
                     "s"(__builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)(lds + 1024 * n))) : "memory");
    }
}
// this wavefront's copies have landed, and behind the barrier everyone's; and everyone is done with what was read before it
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// N fragments, each read from LDS while the products of the one before it run; the barrier keeps the compiler from reading
// them all at once, for which there are no registers
template <int N, bool AHEAD = true, typename Read, typename Use>
__device__ __forceinline__ void pipelined(Read read, Use use) {
    u32x4 f[AHEAD ? 2 : 1][kPlanes];
    if (AHEAD) read(0, f[0]);
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (!AHEAD) read(i, f[0]);
        else if (i + 1 < N) read(i + 1, f[(i + 1) & 1]);
        use(i, f[AHEAD ? i & 1 : 0]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// eight of a lane's accumulators, contraction step s of the next product
__device__ __forceinline__ void accumulator_fragment(const f32x16& a, int s, u32x4 (&f)[kPlanes]) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = a[8 * s + e];
    split_eight(x, f);
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; e++) z[e] = 0.f;
    return z;
}

// scores of a block [32 keys as rows][32 queries as columns] in log2 units: scaled, biased, masked.  rel0 = first key - first
// query position; keys_left = valid keys from the block's first on.  Returns the bucket all of it falls into, or -1
__device__ __forceinline__ int finish_scores(const RelArgs& g, const Bias& bias, f32x16& s, float c, int rel0, int keys_left, int wave, int lane) {
    const int constant = constant_bucket(g.b, rel0 - 31, rel0 + 31);
    if (constant >= 0) {
        const float t = constant == g.b.side - 1 ? bias.before : bias.behind;
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = fmaf(s[e], c, t);
    } else {
        const float* w = bias.diagonals(g.b, rel0, wave, lane) + 31 - (lane & 31) + 4 * (lane >> 5);
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = fmaf(s[e], c, w[8 * (e >> 2) + (e & 3)]);
    }
    if (keys_left < 32 || (g.causal && rel0 + 31 > 0)) {
        // a key is seen when its row is below keys_left and, causal, rel0 + row - column <= 0
        int lim = min(keys_left, 32);
        if (g.causal) lim = min(lim, (lane & 31) - rel0 + 1);
        const int own = lim - 4 * (lane >> 5);
#pragma unroll
        for (int e = 0; e < 16; e++)
            if (8 * (e >> 2) + (e & 3) >= own) s[e] = -INFINITY;
    }
    return constant;
}

// workgroup number -> (batch*head, tile): a head's tiles stay on one XCD, whose L2 then holds its keys and values.  Tiles of one
// length go head by head.  Under a causal mask (`falling`) all the heads' longest tiles (the last) come first and the shorter ones
// fill up behind them: head by head the last head's longest tile would start when the others are nearly done.
__device__ __forceinline__ void head_and_tile(int id, int heads, int tiles, bool falling, int& bh, int& tile) {
    const int xcds = heads % kNumXcd == 0 ? kNumXcd : 1, x = id % xcds, j = id / xcds, per = heads / xcds;
    bh = x + xcds * (falling ? j % per : j / tiles);
    tile = tiles - 1 - (falling ? j / per : j % tiles);
}

constexpr int kThreads = 256, kWaves = 4, kQueryTile = 128;

// ---------------------------------------------------------------------------------------------------- forward
// A row's results: a part of it (splits), or the output and the log-sum-exp.  l: the whole row's sum; o: a lane's accumulators
template <int DP>
__device__ __forceinline__ void store_forward(const RelArgs& g, const f32x16 (&o)[DP / 32], float m, float l, int bh, int64_t qi, int split, int lane) {
    const int64_t row = (int64_t)bh * g.sq + qi;
    float* dst;
    float f = 1.f;
    bool vec = g.vec_o;
    if (g.splits > 1) {
        const int64_t at = (int64_t)split * g.batch * g.heads * g.sq + row;
        dst = g.part_o + at * g.d;
        vec = g.d % 4 == 0;
        if (lane < 32) { g.part_ml[2 * at] = m; g.part_ml[2 * at + 1] = l; }
    } else {
        dst = g.out + bh / g.heads * g.os[0] + bh % g.heads * g.os[1] + qi * g.os[2];
        // a row that sees nothing has the sum 0 and is zero; one whose scores are NaN has no maximum either, but the sum NaN
        f = l == 0.f ? 0.f : 1.f / l;
        if (lane < 32) g.lse[row] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
    }
#pragma unroll
    for (int b = 0; b < DP / 32; b++)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int cd = 32 * b + acc_row(e, lane);
            f32x4 y;
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = o[b][e + j] * f;
            if (vec && cd + 4 <= g.d) *reinterpret_cast<f32x4*>(dst + cd) = y;
            else
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (cd + j < g.d) dst[cd + j] = y[j];
        }
}

// one block of 32 keys (or two) into the running softmax: scores become probabilities, the sums of before are rescaled
template <int NB, int ND>
__device__ __forceinline__ void running_softmax(f32x16 (&s)[NB], float& m, float& l, f32x16 (&o)[ND]) {
    float top = m;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) top = fmaxf(top, s[b][e]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float base = top == -INFINITY ? 0.f : top;                          // nothing seen yet
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    m = top;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            s[b][e] = __builtin_amdgcn_exp2f(s[b][e] - base);
            sum += s[b][e];
        }
    l = l * alpha + sum;
    if (__any(alpha != 1.f)) {
#pragma unroll
        for (int b = 0; b < ND; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[b][e] *= alpha;
    }
}

template <int DP> struct ForwardLds {
    static constexpr int NB = DP <= 64 ? 2 : 1;                               // blocks of 32 keys a step
    static constexpr int V = NB * Block<DP>::BYTES;
    static constexpr int BIAS = 2 * V;
    static constexpr int BYTES = BIAS + Bias::BYTES;
};

// A workgroup owns 128 queries of a head, a wavefront 32 of them, and walks over the keys.  Keys and values have a place in
// LDS each: the next keys are on their way while the values are worked on and the other way round.  Bound by the matrix cores and
// the exponentials and splits beside them (matrix cores busy for 61 % of the cycles): 128 heads of 1024 x 1024 at head size 64 180 us, 190 TFLOP/s of fp32 products (a large
// library product in bf16 has 195 to offer at six products each), causal 121 us.
template <int DP>
__global__ __launch_bounds__(kThreads, 2) void relattn_forward_kernel(RelArgs g) {
    using L = ForwardLds<DP>;
    constexpr int NB = L::NB, KEYS = 32 * NB, ND = DP / 32, KD = DP / 16;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int bh, tile;
    head_and_tile(blockIdx.x, g.batch * g.heads, g.q_tiles, g.causal, bh, tile);
    const int bt = bh / g.heads, h = bh % g.heads, hk = h / g.group;
    const float* q = g.q + bt * g.qs[0] + h * g.qs[1];
    const int64_t plane0 = ((int64_t)bt * g.kv_heads + hk) * g.k_blocks * Block<DP>::BYTES;
    const char *kp = g.k_row + plane0, *vp = g.v_col + plane0;
    const Bias bias(g, h, smem + L::BIAS, kThreads);

    const int q0 = tile * kQueryTile, qw = q0 + 32 * wave;                    // this wavefront's queries: qw + 0..31
    const int qi = qw + (lane & 31);
    const int len = length_of(g, bt);
    const int64_t offset = offset_of(g, len);
    int seen = len;                                                           // keys that some query of the workgroup sees
    if (g.causal) seen = (int)min((int64_t)seen, max((int64_t)0, min((int64_t)q0 + kQueryTile, g.sq) + offset));
    const int kb = (int)min((int64_t)seen, blockIdx.y * g.keys_per_split), ke = (int)min((int64_t)seen, kb + g.keys_per_split);
    const int rel_q = (int)(qw + offset);                                   // position of the wavefront's first query
    if (kb < ke) {
        copy_to_lds<2 * NB * DP * 96 / 1024, kWaves>(kp + (int64_t)(kb / 32) * Block<DP>::BYTES, smem, wave, lane);
    }
    u32x4 qf[KD][kPlanes];
#pragma unroll
    for (int s = 0; s < KD; s++) {
        float x[8];
        row_eight(q + min((int64_t)qi, g.sq - 1) * g.qs[2], true, 16 * s + 8 * (lane >> 5), g.d, g.vec_q, x);
        split_eight<true>(x, qf[s]);
    }
    f32x16 o[ND];
#pragma unroll
    for (int b = 0; b < ND; b++) o[b] = zero16();
    float m = -INFINITY, l = 0.f;
    const float c = g.scale * kLog2e;
    wait_copies();
    int k0 = kb;
    asm volatile("" : "+s"(k0));                                              // keeps the fragments' making apart from the steps
    for (; k0 < ke; k0 += KEYS) {
        copy_to_lds<2 * NB * DP * 96 / 1024, kWaves>(vp + (int64_t)(k0 / 32) * Block<DP>::BYTES, smem + L::V, wave, lane);
        const bool mine = qw < g.sq && !(g.causal && k0 > rel_q + 31);        // else nothing here for this wavefront
        f32x16 s[NB];
        if (mine) {
#pragma unroll
            for (int b = 0; b < NB; b++) s[b] = zero16();
            pipelined<NB * KD>([&](int i, u32x4 (&a)[kPlanes]) { Block<DP>::row_fragment(smem + i / KD * Block<DP>::BYTES, i % KD, lane, a); },
                               [&](int i, const u32x4 (&a)[kPlanes]) { s[i / KD] = mfma_split(a, qf[i % KD], s[i / KD]); });
        }
        wait_copies();
        if (k0 + KEYS < ke)
            copy_to_lds<2 * NB * DP * 96 / 1024, kWaves>(kp + (int64_t)((k0 + KEYS) / 32) * Block<DP>::BYTES, smem, wave, lane);
        if (mine) {
#pragma unroll
            for (int b = 0; b < NB; b++) finish_scores(g, bias, s[b], c, k0 + 32 * b - rel_q, ke - k0 - 32 * b, wave, lane);
            running_softmax(s, m, l, o);
            u32x4 p[kPlanes];
            pipelined<2 * NB * ND>([&](int i, u32x4 (&a)[kPlanes]) {
                                       Block<DP>::column_fragment(smem + L::V + i / ND / 2 * Block<DP>::BYTES, i % ND, i / ND % 2, lane, a);
                                   },
                                   [&](int i, const u32x4 (&a)[kPlanes]) {
                                       if (i % ND == 0) accumulator_fragment(s[i / ND / 2], i / ND % 2, p);
                                       o[i % ND] = mfma_split(a, p, o[i % ND]);
                                   });
        }
        wait_copies();
    }
    if (qi >= g.sq) return;
    l += __shfl_xor(l, 32, 64);
    store_forward<DP>(g, o, m, l, bh, qi, blockIdx.y, lane);
}

// ---- few query rows (of all the heads that share a key head together) over many keys: wavefronts split the keys, each reads
// its keys and values once, straight into fragments.  One query of 64 heads over 8001 keys (262 MB), with joining: 57 us where
// the memory-side cache holds what it can of them from the call before, 67 us (3.9 TB/s) where it holds nothing.
constexpr int kRowWaves = 4;
template <int DP>
__global__ __launch_bounds__(64 * kRowWaves, DP <= 96 ? 2 : 1) void relattn_rows_kernel(RelArgs g, int row_tiles) {
    constexpr int ND = DP / 32, KD = DP / 16;
    __shared__ int border[kMaxBuckets / 2 + 4];
    __shared__ float ml[kRowWaves][2][32];
    __shared__ float part[kRowWaves][32][33];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Each sequence's own keys are cut evenly, and the sequences take turns from part to part: the workgroups that share a compute
    // unit (half a launch apart) then belong to a long and a short one (16 heads, lengths 8001, 5490, 4569, 5989, one
    // call after the other, 47 us against 52).
    const int rt = blockIdx.x % row_tiles, bk = blockIdx.x / row_tiles, hk = bk % g.kv_heads;
    const int bt = (bk / g.kv_heads + (int)((int64_t)blockIdx.y * g.batch / g.splits)) % g.batch;
    const int rows = g.group * (int)g.sq, r = min(32 * rt + (lane & 31), rows - 1);
    const int h = hk * g.group + r / (int)g.sq, qi = r % (int)g.sq;            // this lane's row
    const float* k = g.k + bt * g.ks[0] + hk * g.ks[1];
    const float* v = g.v + bt * g.vs[0] + hk * g.vs[1];
    for (int i = tid; i <= g.b.far; i += 64 * kRowWaves) border[i] = g.b.border[i];
    __syncthreads();
    const int len = length_of(g, bt);
    const int64_t offset = offset_of(g, len);
    const int seen = g.causal ? (int)max((int64_t)0, min((int64_t)len, g.sq + offset)) : len;
    const int unit = 32 * kRowWaves, per = ((seen + unit - 1) / unit + g.splits - 1) / g.splits * unit;
    const int kb = (int)min((int64_t)seen, (int64_t)blockIdx.y * per), ke = (int)min((int64_t)seen, (int64_t)kb + per);
    const int pos = (int)(qi + offset);
    u32x4 qf[KD][kPlanes];
#pragma unroll
    for (int s = 0; s < KD; s++) {
        float x[8];
        row_eight(g.q + bt * g.qs[0] + h * g.qs[1] + qi * g.qs[2], true, 16 * s + 8 * (lane >> 5), g.d, g.vec_q, x);
        split_eight<true>(x, qf[s]);
    }
    f32x16 o[ND];
#pragma unroll
    for (int b = 0; b < ND; b++) o[b] = zero16();
    float m = -INFINITY, l = 0.f;
    const float c = g.scale * kLog2e;
    for (int k0 = kb + 32 * wave; k0 < ke; k0 += 32 * kRowWaves) {
        // a lane's key of the block, and its eight keys of each step of the second product; past the end the last key is read
        // and does not count
        const float* kr = k + (int64_t)min(k0 + (lane & 31), ke - 1) * g.ks[2];
        float x[KD][8], y[2][ND][8];
#pragma unroll
        for (int s = 0; s < KD; s++) row_eight(kr, true, 16 * s + 8 * (lane >> 5), g.d, g.vec_k, x[s]);
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float* vr = v + (int64_t)min(k0 + 16 * s + 4 * (lane >> 5) + (e < 4 ? e : e + 4), ke - 1) * g.vs[2];
#pragma unroll
                for (int b = 0; b < ND; b++) y[s][b][e] = vr[min(32 * b + (lane & 31), g.d - 1)];
            }
        f32x16 s[1] = {zero16()};
#pragma unroll
        for (int t = 0; t < KD; t++) {
            u32x4 a[kPlanes];
            split_eight<true>(x[t], a);
            s[0] = mfma_split(a, qf[t], s[0]);
        }
        const int rel0 = k0 - pos;                                            // the block's first key as this row sees it
        const int constant = constant_bucket(g.b, rel0, rel0 + 31);
        if (__all(constant >= 0)) {
            const float t = table_value(g, constant, h);
#pragma unroll
            for (int e = 0; e < 16; e++) s[0][e] = fmaf(s[0][e], c, t);
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) s[0][e] = fmaf(s[0][e], c, table_value(g, bucket_of(g.b, border, rel0 + acc_row(e, lane)), h));
        }
        int lim = ke - k0;
        if (g.causal) lim = min(lim, 1 - rel0);
        lim -= 4 * (lane >> 5);
        if (__any(lim < 32)) {
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (8 * (e >> 2) + (e & 3) >= lim) s[0][e] = -INFINITY;
        }
        running_softmax(s, m, l, o);
#pragma unroll
        for (int t = 0; t < 2; t++) {
            u32x4 p[kPlanes];
            accumulator_fragment(s[0], t, p);
#pragma unroll
            for (int b = 0; b < ND; b++) {
                u32x4 a[kPlanes];
                split_eight<true>(y[t][b], a);
                o[b] = mfma_split(a, p, o[b]);
            }
        }
    }
    // the wavefronts' parts: 32 of d at a time through LDS
    l += __shfl_xor(l, 32, 64);
    if (lane < 32) { ml[wave][0][lane] = m; ml[wave][1][lane] = l; }
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWaves; w++) top = fmaxf(top, ml[w][0][lane & 31]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kRowWaves; w++) sum += ml[w][1][lane & 31] * __builtin_amdgcn_exp2f(ml[w][0][lane & 31] - base);
    const float own = __builtin_amdgcn_exp2f(m - base);
#pragma unroll
    for (int b = 0; b < ND; b++) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; e++) part[wave][acc_row(e, lane)][lane & 31] = own == 0.f ? 0.f : o[b][e] * own;
        __syncthreads();
        if (wave == 0)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                float t = 0.f;
#pragma unroll
                for (int w = 0; w < kRowWaves; w++) t += part[w][acc_row(e, lane)][lane & 31];
                o[b][e] = t;
            }
    }
    if (wave == 0 && 32 * rt + (lane & 31) < rows) store_forward<DP>(g, o, top, sum, bt * g.heads + h, qi, blockIdx.y, lane);
}

// the splits' parts of a row: 16 lanes a row, which hold the weights of at most 64 splits
__global__ __launch_bounds__(256) void relattn_join_kernel(RelArgs g) {
    const int64_t rows = (int64_t)g.batch * g.heads * g.sq, mine = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int64_t row = min(mine, rows - 1);
    const int lane = threadIdx.x & 15;
    float m[4], l[4], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        m[i] = -INFINITY;
        l[i] = 0.f;
        if (lane + 16 * i < g.splits) {
            const f32x2 ml = *reinterpret_cast<const f32x2*>(g.part_ml + 2 * ((lane + 16 * i) * rows + row));
            m[i] = ml[0];
            l[i] = ml[1];
        }
        top = fmaxf(top, m[i]);
    }
#pragma unroll
    for (int x = 1; x < 16; x *= 2) top = fmaxf(top, __shfl_xor(top, x, 64));
    const float base = top == -INFINITY ? 0.f : top;
    float w[4], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w[i] = __builtin_amdgcn_exp2f(m[i] - base);                           // 0 where there is no split
        sum += l[i] * w[i];
    }
#pragma unroll
    for (int x = 1; x < 16; x *= 2) sum += __shfl_xor(sum, x, 64);
    const int64_t bh = row / g.sq, qi = row - bh * g.sq, bt = bh / g.heads, h = bh - bt * g.heads;
    float* dst = g.out + bt * g.os[0] + h * g.os[1] + qi * g.os[2];
    const float f = sum == 0.f ? 0.f : 1.f / sum;                             // as in store_forward
    const bool vec = g.d % 4 == 0;
    for (int c0 = 0; c0 < g.d; c0 += 64) {
        const int c = c0 + 4 * lane, n = min(4, g.d - c), at = min(c, g.d - 1) & (vec ? ~3 : ~0);
        const float* p = g.part_o + row * g.d + at;
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < g.splits; s0 += 4) {                            // four loads at a time; past the last split weight 0
            f32x4 x[4];
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const float* from = p + min(s0 + s, g.splits - 1) * rows * g.d;
                if (vec) x[s] = *reinterpret_cast<const f32x4*>(from);
                else
#pragma unroll
                    for (int j = 0; j < 4; j++) x[s][j] = from[max(0, min(j, n - 1))];
            }
            const int i = s0 >> 4;
            const float ws = i == 0 ? w[0] : i == 1 ? w[1] : i == 2 ? w[2] : w[3];
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const float y = __shfl(ws, (threadIdx.x & 48) + ((s0 + s) & 15), 64);
#pragma unroll
                for (int j = 0; j < 4; j++) a[j] += y == 0.f ? 0.f : y * x[s][j];
            }
        }
        if (mine < rows && n > 0) {
#pragma unroll
            for (int j = 0; j < 4; j++) a[j] *= f;
            if (g.vec_o) *reinterpret_cast<f32x4*>(dst + c) = a;
            else
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (j < n) dst[c + j] = a[j];
        }
    }
    if (mine < rows && lane == 0) g.lse[row] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// ---------------------------------------------------------------------------------------------------- backward
// The kernel's arguments read anew, where a walk is over: kept from its start on they would hold scalar registers through it
// (they are the kernel's first parameter).
using Arguments = const __attribute__((address_space(4))) RelArgs;
__device__ __forceinline__ Arguments* arguments_again() {
    Arguments* a = (Arguments*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return a;
}
// log2 e * lse; rows that see nothing get a number (their scores are all masked)
__device__ __forceinline__ float lse_log2(float lse) { return lse == -INFINITY ? 0.f : lse * kLog2e; }

template <int DP> struct QueryLds {
    static constexpr int V = Block<DP>::BYTES, KT = 2 * Block<DP>::BYTES;     // keys and values in row form, keys in column form
    static constexpr int BIAS = 3 * Block<DP>::BYTES;
    static constexpr int SUMS = BIAS + Bias::BYTES;                           // per wavefront: a sum per bucket, in 64 bits
    static constexpr int BLOCK = SUMS + kWaves * kMaxBuckets * 8;             // per wavefront: a block of dS, rows of 33
    static constexpr int BYTES = BLOCK + kWaves * 32 * 33 * 4;
};

// dQ and the table's gradient: a workgroup owns 128 queries of a head and walks over the keys
template <int DP>
__device__ __forceinline__ void query_tile(const RelArgs& g, int id, int part) {
    using L = QueryLds<DP>;
    constexpr int KEYS = 32, ND = DP / 32, KD = DP / 16, KB = Block<DP>::BYTES / 1024;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    double* sums = reinterpret_cast<double*>(smem + L::SUMS) + kMaxBuckets * wave;
    float* block = reinterpret_cast<float*>(smem + L::BLOCK) + 32 * 33 * wave;
    int bh, tile;
    head_and_tile(id, g.batch * g.heads, g.q_tiles, g.causal, bh, tile);
    const int bt = bh / g.heads, h = bh % g.heads, hk = h / g.group;
    const float* q = g.q + bt * g.qs[0] + h * g.qs[1];
    const float* dout = g.d_out + bt * g.os[0] + h * g.os[1];
    const int64_t plane0 = ((int64_t)bt * g.kv_heads + hk) * g.k_blocks * Block<DP>::BYTES;
    const Bias bias(g, h, smem + L::BIAS, kThreads);
    for (int i = lane; i < g.buckets; i += 64) sums[i] = 0.0;

    const int q0 = tile * kQueryTile, qw = q0 + 32 * wave, qi = qw + (lane & 31);
    const bool live = qi < g.sq;
    const int len = length_of(g, bt);
    const int64_t offset = offset_of(g, len);
    int ke = len;
    if (g.causal) ke = (int)min((int64_t)ke, max((int64_t)0, min((int64_t)q0 + kQueryTile, g.sq) + offset));
    const int kb = (int)(part * g.keys_per_split);
    ke = (int)min((int64_t)ke, kb + g.keys_per_split);
    const int rel_q = (int)(qw + offset);
    const auto fetch_rows = [&](int k0) {
        const int64_t at = plane0 + (int64_t)(k0 / 32) * Block<DP>::BYTES;
        copy_to_lds<KB, kWaves>(g.k_row + at, smem, wave, lane);
        copy_to_lds<KB, kWaves>(g.v_row + at, smem + L::V, wave, lane);
    };
    if (kb < ke) fetch_rows(kb);
    // The matrix cores' sums are cut towards minus infinity by some hundredths of a step.  For one element that is nothing, but
    // the table's gradient adds up a million of them that nearly cancel: odd queries are negated, and their results again, so
    // that the cuts cancel too (8 x 16 heads x 1024 x 1024: the table's relative error 4e-6 without, 4e-7 with it).
    const float sign = lane & 1 ? -1.f : 1.f;
    u32x4 qf[KD][kPlanes], gf[KD][kPlanes];
    const int64_t qrow = min((int64_t)qi, g.sq - 1);
#pragma unroll
    for (int s = 0; s < KD; s++) {
        float x[8];
        row_eight(q + qrow * g.qs[2], live, 16 * s + 8 * (lane >> 5), g.d, g.vec_q, x);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= sign;
        split_eight<true>(x, qf[s]);
        row_eight(dout + qrow * g.os[2], live, 16 * s + 8 * (lane >> 5), g.d, g.vec_o, x);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= sign;
        split_eight<true>(x, gf[s]);
    }
    const int64_t row = (int64_t)bh * g.sq + qrow;
    const float lse = lse_log2(g.lse_in[row]), delta = g.delta[row];
    const float c = g.scale * kLog2e * sign;
    f32x16 dq[ND];
#pragma unroll
    for (int b = 0; b < ND; b++) dq[b] = zero16();
    // A bucket's sum is small against its terms (a row of dS adds up to zero): blocks are added up in 64 bits
    double far_sum[2] = {0.0, 0.0};                                           // blocks that lie in one bucket: before, behind
    wait_copies();
    int k0 = kb;
    asm volatile("" : "+s"(k0));                                              // keeps the fragments' making apart from the steps
    for (; k0 < ke; k0 += KEYS) {
        copy_to_lds<KB, kWaves>(g.k_col + plane0 + (int64_t)(k0 / 32) * Block<DP>::BYTES, smem + L::KT, wave, lane);
        const bool mine = qw < g.sq && !(g.causal && k0 > rel_q + 31);
        f32x16 s, dp;
        if (mine) {
            s = zero16();
            dp = zero16();
            pipelined<2 * KD>([&](int i, u32x4 (&a)[kPlanes]) { Block<DP>::row_fragment(smem + (i & 1 ? L::V : 0), i >> 1, lane, a); },
                              [&](int i, const u32x4 (&a)[kPlanes]) {
                                  if (i & 1) dp = mfma_split(a, gf[i >> 1], dp);
                                  else s = mfma_split(a, qf[i >> 1], s);
                              });
        }
        wait_copies();
        if (k0 + KEYS < ke) fetch_rows(k0 + KEYS);
        if (mine) {
        const int constant = finish_scores(g, bias, s, c, k0 - rel_q, ke - k0, wave, lane);
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = live ? __builtin_amdgcn_exp2f(s[e] - lse) * fmaf(dp[e], sign, -delta) : 0.f;
        if (constant >= 0) {
            float t[8];
#pragma unroll
            for (int e = 0; e < 8; e++) t[e] = s[e] + s[8 + e];
            const double all = (double)((t[0] + t[1]) + (t[2] + t[3])) + (double)((t[4] + t[5]) + (t[6] + t[7]));
            if (constant == g.b.side - 1) far_sum[0] += all; else far_sum[1] += all;
        } else {
            // diagonal `lane` of the block: key row r, query column x with r - x = lane - 31
            const int bucket = bias.bucket(g.b, k0 - rel_q + lane - 31);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int e = 0; e < 16; e++) block[acc_row(e, lane) * 33 + (lane & 31)] = s[e];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            double t = 0.0;
#pragma unroll 2
            for (int x0 = 0; x0 < 32; x0 += 8) {
                float part[8];
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const int r = lane - 31 + x0 + x;
                    const float y = block[min(max(r, 0), 31) * 33 + x0 + x];
                    part[x] = r >= 0 && r < 32 ? y : 0.f;
                }
                t += (double)((part[0] + part[1]) + (part[2] + part[3])) + (double)((part[4] + part[5]) + (part[6] + part[7]));
            }
            // lanes of one bucket are neighbours: sums of runs, the last lane of a run adds it to the bucket
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const double y = __shfl_up(t, off, 64);
                const int other = __shfl_up(bucket, off, 64);
                if (lane >= off && other == bucket) t += y;
            }
            const int after = __shfl_down(bucket, 1, 64);
            if (lane == 63 || after != bucket) sums[bucket] += t;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        u32x4 p[kPlanes];
        pipelined<2 * ND>([&](int i, u32x4 (&a)[kPlanes]) { Block<DP>::column_fragment(smem + L::KT, i % ND, i / ND, lane, a); },
                          [&](int i, const u32x4 (&a)[kPlanes]) {
                              if (i % ND == 0) accumulator_fragment(s, i / ND, p);
                              dq[i % ND] = mfma_split(a, p, dq[i % ND]);
                          });
        }
        wait_copies();
    }
    far_sum[0] = wave_sum_f64(far_sum[0]);
    far_sum[1] = wave_sum_f64(far_sum[1]);
    if (lane == 0) {
        sums[g.b.side - 1] += far_sum[0];
        sums[g.b.both ? 2 * g.b.side - 1 : 0] += far_sum[1];
    }
    __syncthreads();
    const double* all = reinterpret_cast<const double*>(smem + L::SUMS);
    const int64_t split_bh = (int64_t)part * g.batch * g.heads;
    for (int i = tid; i < g.buckets; i += kThreads)
        g.part_table[((split_bh + bh) * g.q_tiles + tile) * g.buckets + i] =
            (all[i] + all[kMaxBuckets + i]) + (all[2 * kMaxBuckets + i] + all[3 * kMaxBuckets + i]);
    if (!live) return;
    Arguments& e = *arguments_again();
    const bool parts = e.splits > 1, vec = parts ? e.d % 4 == 0 : e.vec_q;
    float* dst = parts ? e.part_q + ((split_bh + bh) * e.sq + qi) * e.d : e.dq + bt * e.qs[0] + h * e.qs[1] + qi * e.qs[2];
#pragma unroll
    for (int b = 0; b < DP / 32; b++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int cd = 32 * b + acc_row(r, lane);
            f32x4 y;
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = dq[b][r + j] * e.scale;
            if (vec && cd + 4 <= e.d) *reinterpret_cast<f32x4*>(dst + cd) = y;
            else
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (cd + j < e.d) dst[cd + j] = y[j];
        }
}

template <int DP> struct KeyLds {
    static constexpr int G = Block<DP>::BYTES;                                // queries and dO: row form, then column form
    static constexpr int QT = 2 * G, GT = 3 * G;
    static constexpr int STAT = 4 * G;                                        // lse and delta of a step's queries, twice
    static constexpr int BIAS = STAT + 2 * 64 * 4;
    static constexpr int BYTES = BIAS + Bias::BYTES;
};

// dK and dV of one query head: a workgroup owns 128 keys and walks over the queries.  Heads that share a key head leave their
// parts in work memory (one long chain of sums over all of them would round more, and fill fewer compute units)
template <int DP>
__device__ __forceinline__ void key_tile(const RelArgs& g, int id, int part) {
    using L = KeyLds<DP>;
    constexpr int ROWS = 32, ND = DP / 32, KD = DP / 16, KB = Block<DP>::BYTES / 1024;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int bh, tile;
    const int k_tiles = (int)((g.sk + 127) / 128);
    head_and_tile(id, g.batch * g.heads, k_tiles, g.causal, bh, tile);
    tile = k_tiles - 1 - tile;                                                // the first keys are seen by the most queries
    const int bt = bh / g.heads, h = bh % g.heads, hk = h / g.group;
    const float* k = g.k + bt * g.ks[0] + hk * g.ks[1];
    const float* v = g.v + bt * g.vs[0] + hk * g.vs[1];
    const int kw = tile * 128 + 32 * wave, ki = kw + (lane & 31), sq = (int)g.sq;
    const int len = length_of(g, bt);
    const int64_t offset = offset_of(g, len);
    const bool live = ki < len;
    u32x4 kf[KD][kPlanes], vf[KD][kPlanes];
#pragma unroll
    for (int s = 0; s < KD; s++) {
        float x[8];
        row_eight(k + min((int64_t)ki, g.sk - 1) * g.ks[2], live, 16 * s + 8 * (lane >> 5), g.d, g.vec_k, x);
        split_eight<true>(x, kf[s]);
        row_eight(v + min((int64_t)ki, g.sk - 1) * g.vs[2], live, 16 * s + 8 * (lane >> 5), g.d, g.vec_v, x);
        split_eight<true>(x, vf[s]);
    }
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int b = 0; b < ND; b++) { dk[b] = zero16(); dv[b] = zero16(); }
    const float c = g.scale * kLog2e;
    int qb = 0;                                                               // causal: the first query that sees a key of the workgroup
    if (g.causal) qb = (int)(min((int64_t)sq, max((int64_t)0, (int64_t)tile * 128 - offset)) / ROWS * ROWS);
    const int qe = min(sq, (part + 1) * g.queries_per_split);
    qb = max(qb, part * g.queries_per_split);
    if (tile * 128 >= len) qb = sq;                                           // only padding here
    // One turn of a loop that the compiler cannot see to be one: it then keeps the fragments' making apart from the steps.
    // Run together they need 47 registers more than there are at head size 128.
    int turns = 1;
    asm volatile("" : "+s"(turns));
    for (; turns > 0 && qb < qe; turns--) {
        const int64_t row0 = (int64_t)bh * g.sq, plane0 = (int64_t)bh * g.q_blocks * Block<DP>::BYTES;
        const auto fetch = [&](const char* q, const char* d, int r0, int at) {
            const int64_t o = plane0 + (int64_t)(r0 / 32) * Block<DP>::BYTES;
            copy_to_lds<KB, kWaves>(q + o, smem + at, wave, lane);
            copy_to_lds<KB, kWaves>(d + o, smem + at + L::G, wave, lane);
        };
        const auto fetch_stat = [&](int r0, int buffer) {
            if (tid < 2 * ROWS) {
                const int r = min(r0 + (tid & (ROWS - 1)), sq - 1);
                reinterpret_cast<float*>(smem + L::STAT)[64 * buffer + tid] = tid < ROWS ? lse_log2(g.lse_in[row0 + r]) : g.delta[row0 + r];
            }
        };
        const Bias bias(g, h, smem + L::BIAS, kThreads);
        // from the last queries down: under a causal mask, where the key tiles have different first queries, all the workgroups
        // of a head are then at the same queries at the same time and read them out of the L2 once
        const int q_last = (qe - 1) / ROWS * ROWS;
        fetch(g.q_row, g.g_row, q_last, 0);
        fetch_stat(q_last, 0);
        wait_copies();
        for (int r0 = q_last, turn = 0; r0 >= qb; r0 -= ROWS, turn ^= 1) {
            fetch(g.q_col, g.g_col, r0, L::QT);
            if (r0 > qb) fetch_stat(r0 - ROWS, turn ^ 1);
            const float* stat = reinterpret_cast<const float*>(smem + L::STAT) + 64 * turn;
            const bool mine = kw < len && !(g.causal && kw > min(r0 + ROWS, sq) - 1 + offset);
            f32x16 s, dp;
            if (mine) {
                s = zero16();
                dp = zero16();
                pipelined<2 * KD>([&](int i, u32x4 (&a)[kPlanes]) { Block<DP>::row_fragment(smem + (i & 1 ? L::G : 0), i >> 1, lane, a); },
                                  [&](int i, const u32x4 (&a)[kPlanes]) {
                                      if (i & 1) dp = mfma_split(a, vf[i >> 1], dp);
                                      else s = mfma_split(a, kf[i >> 1], s);
                                  });
            }
            wait_copies();
            if (r0 > qb) fetch(g.q_row, g.g_row, r0 - ROWS, 0);
            if (mine) {
            // block [32 queries as rows][32 keys as columns]
            const int rel0 = (int)(kw - r0 - offset);
            const int constant = constant_bucket(g.b, rel0 - 31, rel0 + 31);
            const f32x4* ls = reinterpret_cast<const f32x4*>(stat + 4 * (lane >> 5));   // lse of rows 8g + 4 half + 0..3
            if (constant >= 0) {
                const float t = constant == g.b.side - 1 ? bias.before : bias.behind;
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] = fmaf(s[e], c, t - ls[2 * (e >> 2)][e & 3]);
            } else {
                const float* w = bias.diagonals(g.b, rel0, wave, lane) + (lane & 31) - 4 * (lane >> 5) + 4;
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] = fmaf(s[e], c, w[27 - 8 * (e >> 2) - (e & 3)] - ls[2 * (e >> 2)][e & 3]);
            }
            // a query sees the key when the key is valid, the query is one and, causal, rel0 + column - row <= 0
            const int half4 = 4 * (lane >> 5);
            const int first = (g.causal ? rel0 + (lane & 31) : 0) - half4, last = (live ? min(ROWS, sq - r0) : 0) - half4;
            const bool masks = kw + 32 > len || r0 + ROWS > sq || (g.causal && rel0 + 31 > 0);
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = __builtin_amdgcn_exp2f(s[e]);
            if (masks) {
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int r = 8 * (e >> 2) + (e & 3);
                    if (r < first || r >= last) s[e] = 0.f;
                }
            }
            const f32x4* dl = reinterpret_cast<const f32x4*>(stat + ROWS + 4 * (lane >> 5));
#pragma unroll
            for (int e = 0; e < 16; e++) dp[e] = s[e] * (dp[e] - dl[2 * (e >> 2)][e & 3]);
            u32x4 x[kPlanes];
            pipelined<4 * ND, DP != 64>([&](int i, u32x4 (&a)[kPlanes]) {
                                  Block<DP>::column_fragment(smem + (i < 2 * ND ? L::GT : L::QT), i % ND, i / ND % 2, lane, a);
                              },
                              [&](int i, const u32x4 (&a)[kPlanes]) {
                                  if (i % ND == 0) accumulator_fragment(i < 2 * ND ? s : dp, i / ND % 2, x);
                                  if (i < 2 * ND) dv[i % ND] = mfma_split(a, x, dv[i % ND]);
                                  else dk[i % ND] = mfma_split(a, x, dk[i % ND]);
                              });
            }
            wait_copies();
        }
    }
    Arguments& e = *arguments_again();
    int again = threadIdx.x;
    asm volatile("" : "+v"(again));
    const int kj = tile * 128 + again / 64 * 32 + (again & 31);
    if (kj >= e.sk) return;
    const bool parts = e.part_k;
    const int64_t at = (((int64_t)part * e.batch * e.heads + bh) * e.sk + kj) * e.d;
    float* pk = parts ? e.part_k + at : e.dk + bt * e.ks[0] + hk * e.ks[1] + kj * e.ks[2];
    float* pv = parts ? e.part_v + at : e.dv + bt * e.vs[0] + hk * e.vs[1] + kj * e.vs[2];
    const bool vec_k = parts ? e.d % 4 == 0 : e.vec_k, vec_v = parts ? e.d % 4 == 0 : e.vec_v;
#pragma unroll
    for (int b = 0; b < ND; b++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int cd = 32 * b + acc_row(r, again & 63);
            f32x4 x, y;
#pragma unroll
            for (int j = 0; j < 4; j++) { x[j] = dk[b][r + j] * e.scale; y[j] = dv[b][r + j]; }
            if (vec_k && cd + 4 <= e.d) *reinterpret_cast<f32x4*>(pk + cd) = x;
            else
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (cd + j < e.d) pk[cd + j] = x[j];
            if (vec_v && cd + 4 <= e.d) *reinterpret_cast<f32x4*>(pv + cd) = y;
            else
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (cd + j < e.d) pv[cd + j] = y[j];
            __builtin_amdgcn_sched_barrier(0);
        }
}

// Both walks in one launch: the key tiles, which take longer, first, and the query tiles fill up behind them (one launch after the
// other, us: 128 heads of 1024, causal, 482 against 459; 32 heads of 1024 at head size 128 379 against 261).  Bound by the matrix
// cores (49 % of the cycles) at seven products of a head's size, as scores and dP are made in both walks: 128 heads of 1024, causal,
// 420 us, 143 TFLOP/s.  Five products would do, with a part of dQ written for every key tile and the parts added up in order.
template <int DP>
__global__ __launch_bounds__(kThreads, DP <= 64 ? 2 : 1) void relattn_backward_kernel(RelArgs g, int key_groups, int query_groups) {
    const int all_keys = key_groups * g.q_splits, id = blockIdx.x;
    const bool keys = id < all_keys;
    const int at = keys ? id : id - all_keys, groups = keys ? key_groups : query_groups;
    const int part = __builtin_amdgcn_readfirstlane(at / groups), tile = __builtin_amdgcn_readfirstlane(at - part * groups);
    if (keys) key_tile<DP>(g, tile, part);
    else query_tile<DP>(g, tile, part);
}

// n floats (at most 4) of parts that lie `step` apart, `count` of them, added up in order
__device__ __forceinline__ f32x4 sum_of(const float* p, int64_t step, int count, int n, bool vec, f32x4 t) {
    for (int i = 0; i < count; i += 4) {
        f32x4 x[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const float* at = p + min(i + u, count - 1) * step;
            if (vec) x[u] = *reinterpret_cast<const f32x4*>(at);
            else
#pragma unroll
                for (int j = 0; j < 4; j++) x[u][j] = at[min(j, n - 1)];
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int j = 0; j < 4; j++) t[j] += i + u < count ? x[u][j] : 0.f;
    }
    return t;
}
__device__ __forceinline__ void put(float* dst, f32x4 t, int n, bool vec) {
    if (vec) *reinterpret_cast<f32x4*>(dst) = t;
    else
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < n) dst[j] = t[j];
}

// What is left in parts, added up in order: the first workgroups make dT (16 buckets of a head each, over splits, batch and
// tiles), the next ones dQ where the keys were split, the last ones dK and dV where the queries were or heads share a key head;
// 16 or 32 lanes a row, four floats a lane.
struct Fold { int table_blocks, q_blocks, k_blocks; float* dtable; int accumulate; };
__global__ __launch_bounds__(256) void relattn_fold_kernel(RelArgs g, Fold f) {
    __shared__ double red[256];
    const int id = blockIdx.x, lanes = g.d <= 64 ? 16 : 32, c = threadIdx.x % lanes * 4, per_block = 256 / lanes;
    const int n = min(4, g.d - c), slot = threadIdx.x / lanes;
    const bool vec = g.d % 4 == 0;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if (id < f.table_blocks) {
        const int h = id % g.heads, b = id / g.heads * 16 + (threadIdx.x & 15), first = threadIdx.x >> 4;
        const int64_t total = (int64_t)g.splits * g.batch * g.q_tiles;
        double s = 0.0;
        if (b < g.buckets)
            for (int64_t i = first; i < total; i += 16) {
                const int64_t bt = i / g.q_tiles, bh = bt * g.heads + h;
                s += g.part_table[(bh * g.q_tiles + (i - bt * g.q_tiles)) * g.buckets + b];
            }
        red[threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.x < 16 && b < g.buckets) {
            double t = 0.0;
            for (int i = 0; i < 16; i++) t += red[i * 16 + threadIdx.x];
            float* dst = f.dtable + (int64_t)b * g.heads + h;
            *dst = f.accumulate ? *dst + (float)t : (float)t;
        }
    } else if (n <= 0) {
        return;
    } else if (id < f.table_blocks + f.q_blocks) {
        const int64_t rows = (int64_t)g.batch * g.heads * g.sq;
        for (int64_t r = (int64_t)(id - f.table_blocks) * per_block + slot; r < rows; r += (int64_t)f.q_blocks * per_block) {
            const int64_t bh = r / g.sq, row = r - bh * g.sq, bt = bh / g.heads, h = bh - bt * g.heads;
            put(g.dq + bt * g.qs[0] + h * g.qs[1] + row * g.qs[2] + c, sum_of(g.part_q + r * g.d + c, rows * g.d, g.splits, n, vec, zero), n, vec && g.vec_q);
        }
    } else {
        const int64_t rows = (int64_t)g.batch * g.kv_heads * g.sk, per = g.sk * g.d, all = (int64_t)g.batch * g.heads * per;
        for (int64_t r = (int64_t)(id - f.table_blocks - f.q_blocks) * per_block + slot; r < rows; r += (int64_t)f.k_blocks * per_block) {
            const int64_t bk = r / g.sk, row = r - bk * g.sk, bt = bk / g.kv_heads, hk = bk - bt * g.kv_heads;
            const int64_t first = (bt * g.heads + hk * g.group) * per + row * g.d + c;
            f32x4 x = zero, y = zero;
            for (int p = 0; p < g.q_splits; p++) {
                x = sum_of(g.part_k + first + p * all, per, g.group, n, vec, x);
                y = sum_of(g.part_v + first + p * all, per, g.group, n, vec, y);
            }
            put(g.dk + bt * g.ks[0] + hk * g.ks[1] + row * g.ks[2] + c, x, n, vec && g.vec_k);
            put(g.dv + bt * g.vs[0] + hk * g.vs[1] + row * g.vs[2] + c, y, n, vec && g.vec_v);
        }
    }
}

// ---------------------------------------------------------------------------------------------------- host side
// floor(log(n/e) / log(D/e) * far), a distance within 1e-9 of a border counting as past it
static int far_step(int64_t n, int e, int distance, int far) {
    const double t = log((double)n / e) / log((double)distance / e) * far;
    const double f = floor(t + 1e-9);
    return f < 0 ? 0 : f >= far ? far - 1 : (int)f;
}
static bool make_buckets(int num, int distance, int both, Buckets& b) {
    const int side = both ? num / 2 : num, exact = side / 2;
    if (num < 2 || num > kMaxBuckets || (both && num % 2) || exact < 1 || distance <= exact) return false;
    b.both = both ? 1 : 0;
    b.side = side;
    b.exact = exact;
    b.far = side - exact;
    b.log2_exact = (float)log2((double)exact);
    b.per_log2 = (float)(b.far / log2((double)distance / exact));
    b.border[0] = exact;
    for (int j = 1; j < b.far; j++) {
        int64_t n = (int64_t)(exact * pow((double)distance / exact, (double)j / b.far));
        if (n < exact) n = exact;
        while (n > exact && far_step(n - 1, exact, distance, b.far) >= j) n--;
        while (far_step(n, exact, distance, b.far) < j) n++;
        b.border[j] = (int)n;
    }
    b.border[b.far] = 0x7fffffff;
    b.last = b.border[b.far - 1];
    const int64_t line = (b.both ? 2 : 1) * (int64_t)b.last + 128;
    b.line = line <= kLine ? (int)line : 0;
    return true;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool vectors(const void* p, const int64_t (&s)[3], int d) {
    return aligned16(p) && d % 4 == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
}

constexpr int64_t kMostGroups = (1 << 23) - 1;            // workgroups of one launch: their threads are counted in 32 bits

static int relattn_args(const char* fn, const bh_relbias_attention_t* p, RelArgs& g) {
    if (!p) return set_error(BH_EINVAL, "%s: null pointer", fn);
    if (p->batch < 0 || p->heads < 0 || p->kv_heads < 0 || p->sq < 0 || p->sk < 0) return set_error(BH_EINVAL, "%s: negative dimension", fn);
    if (p->d < 1 || p->d > 128) return set_error(BH_EINVAL, "%s: the head size is 1 to 128", fn);
    if (p->heads > 0 && (p->kv_heads < 1 || p->heads % p->kv_heads)) return set_error(BH_EINVAL, "%s: heads is a multiple of kv_heads", fn);
    const int64_t most = (int64_t)1 << 28;                // sums and differences of them (up to five) stay within 32 bits
    if (p->sq > most || p->sk > most || p->query_offset > most || p->query_offset < -most)
        return set_error(BH_EINVAL, "%s: sequences and offset are at most 2^28", fn);
    if (p->batch > 0x7fffffff || p->heads > 0x7fffffff || p->batch * p->heads > 0x7fffffff / 2) return set_error(BH_EINVAL, "%s: too many heads", fn);
    if (p->batch * p->heads > 0 && (ceil_div(p->sq, 32) > 0x3fffffff / (p->batch * p->heads) || ceil_div(p->sk, 32) > 0x3fffffff / (p->batch * p->heads)))
        return set_error(BH_EINVAL, "%s: too many rows", fn);
    for (int i = 0; i < 3; i++)
        if (p->q_stride[i] < 0 || p->k_stride[i] < 0 || p->v_stride[i] < 0 || p->o_stride[i] < 0)
            return set_error(BH_EINVAL, "%s: negative stride", fn);
    if (!make_buckets(p->num_buckets, p->max_distance, p->bidirectional, g.b))
        return set_error(BH_EINVAL, "%s: 2 to %d buckets (4 or more and even for both directions) and a distance past half of a direction's", fn, kMaxBuckets);
    if (!(fabsf(p->scale) < INFINITY)) return set_error(BH_EINVAL, "%s: the scale is a number", fn);
    g.batch = (int)p->batch; g.heads = (int)p->heads; g.kv_heads = (int)p->kv_heads;
    g.group = p->heads ? (int)(p->heads / p->kv_heads) : 1;
    g.d = (int)p->d; g.sq = p->sq; g.sk = p->sk; g.offset = p->query_offset; g.causal = p->causal ? 1 : 0; g.at_end = p->queries_at_end ? 1 : 0; g.scale = p->scale;
    for (int i = 0; i < 3; i++) { g.qs[i] = p->q_stride[i]; g.ks[i] = p->k_stride[i]; g.vs[i] = p->v_stride[i]; g.os[i] = p->o_stride[i]; }
    g.buckets = p->num_buckets;
    g.q_tiles = (int)ceil_div(p->sq, kQueryTile);
    if ((int64_t)g.q_tiles * g.batch * g.heads > kMostGroups || ceil_div(p->sk, 128) * g.batch * g.heads > kMostGroups ||
        ceil_div(g.buckets, 16) * g.heads > kMostGroups)
        return set_error(BH_EINVAL, "%s: too many rows", fn);
    return BH_OK;
}

// outputs that two rows share would be written twice: rows of a head, heads and batch entries must lie apart
static bool rows_apart(const int64_t (&s)[3], int64_t batch, int64_t heads, int64_t rows, int64_t d) {
    struct { int64_t n, s; } v[3] = {{batch, s[0]}, {heads, s[1]}, {rows, s[2]}};
    if (batch == 0 || heads == 0 || rows == 0) return true;
    int64_t extent = d;
    for (int pass = 0; pass < 3; pass++) {
        int at = -1;
        for (int i = 0; i < 3; i++)
            if (v[i].n > 1 && (at < 0 || v[i].s < v[at].s)) at = i;
        if (at < 0) return true;
        if (v[at].s < extent) return false;
        extent = v[at].s * (v[at].n - 1) + extent;
        v[at].n = 1;
    }
    return true;
}

template <typename K>
static int launch_lds(K kernel, bool& raised, dim3 grid, int bytes, const char* what, const RelArgs& g) {
    if (!raised) {
        const int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes), what);
        if (rc) return rc;
        raised = true;
    }
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), bytes, stream(), g);
    return BH_LAUNCH_CHECK(what);
}

// planes of several operands in one launch
struct Planes {
    SplitJobs jobs = {};
    int n = 0;
    int64_t total = 0;
    void add(const float* src, const int64_t (&s)[3], int heads, int batch, int64_t rows, const int32_t* len, int blocks, bool vec, const char* row,
             const char* col) {
        SplitJob& j = jobs.j[n];
        j.src = src; j.heads = heads; j.rows = rows; j.len = len; j.blocks = blocks; j.vec = vec;
        j.row = const_cast<char*>(row); j.col = const_cast<char*>(col);
        for (int i = 0; i < 3; i++) j.s[i] = s[i];
        total += (int64_t)batch * heads * blocks;
        for (int i = ++n; i <= kMaxJobs; i++) jobs.first[i] = (int)(total < kMostGroups ? total : kMostGroups);
    }
    SplitJob& last() { return jobs.j[n - 1]; }
    template <int DP> int launch(int d) {
        if (total > kMostGroups) return set_error(BH_EINVAL, "bh_relbias_attention: too many rows");
        jobs.d = d;
        hipLaunchKernelGGL(relattn_split_kernel<DP>, dim3((unsigned)total), dim3(256), 0, stream(), jobs);
        return BH_LAUNCH_CHECK("bh_relbias_attention: split");
    }
};

static int g_force_rows = -1, g_force_splits = 0;

// Parts into which the walk of `wgs` workgroups is cut, `each` of which share one of the 256 compute units: the longest walk has
// `longest` steps, `mean` is the average.  Where all are alike the rounds of workgroups count, else (longest first) the longest
// walk or all the work spread evenly.  A part's start counts as `start` steps, joining as `join` a part.
// Us whole / in parts as chosen, head size 64: 64 sequences of one query over 8001 keys 187 / 52, 16 heads of 2048 106 / 83; 64
// heads of 256 23 in one part, 39 in two.
static int parts_for(int64_t wgs, int64_t longest, double mean, int each, int start, double join, int most) {
    if (g_force_splits > 0) return (int)(g_force_splits < longest ? g_force_splits : longest > 0 ? longest : 1);
    const int64_t slots = 256 * each;
    int best = 1;
    double least = INFINITY;
    for (int s = 1; s <= most && s <= longest; s++) {
        const double walk = (double)(ceil_div(longest, s) + start), all = (double)(wgs * s) / (double)slots * (mean / s + start);
        const double cost = (mean >= (double)(longest - 1) ? (double)ceil_div(wgs * s, slots) * walk : walk > all ? walk : all) + (s > 1 ? join * (s + 1) : 0.0);
        if (cost < 0.97 * least) { least = cost; best = s; }
    }
    return best;
}
// the pairs of query and key that a causal mask leaves
static double seen_pairs(const RelArgs& g) {
    if (!g.causal) return (double)g.sq * (double)g.sk;
    const int64_t offset = g.at_end ? g.sk - g.sq + g.offset : g.offset;       // as in a sequence of full length
    // query i sees min(max(i + 1 + offset, 0), sk) keys: none below lo, all from hi on
    const int64_t lo = -offset < 0 ? 0 : -offset < g.sq ? -offset : g.sq, full = g.sk - 1 - offset;
    const int64_t hi = full < lo ? lo : full < g.sq ? full : g.sq;
    return ((double)(lo + 1 + offset) + (double)(hi + offset)) * 0.5 * (double)(hi - lo) + (double)(g.sq - hi) * (double)g.sk;
}

template <int DP>
static int run_forward(RelArgs& g) {
    static bool raised = false;
    const int64_t rows = (int64_t)g.batch * g.heads * g.sq;
    const int64_t head_rows = (int64_t)g.group * g.sq, row_tiles = ceil_div(head_rows, 32);
    // The kernel for few rows reads (and splits) the keys once per 32 rows, the tiles need planes made first (us, rows / tiles,
    // head size 64): 64 rows of 128 heads over 4096 keys 112 / 218, 128 rows 193 / 229, of 8 heads 28 / 33, 64 over 128 keys of
    // 96 heads 12 / 20; 128 over 512 keys of 256 heads 64 / 64, over 128 keys of 384 heads 44 / 33, 192 over 192 33 / 24.
    const bool by_rows = g_force_rows >= 0 ? g_force_rows == 1 && head_rows < (1 << 24) : row_tiles <= 2 || (row_tiles <= 4 && g.sk >= 2 * head_rows);
    const int64_t wgs = by_rows ? row_tiles * g.batch * g.kv_heads : (int64_t)g.q_tiles * g.batch * g.heads;
    if (wgs > kMostGroups) return set_error(BH_EINVAL, "bh_relbias_attention_forward: too many rows");
    const int64_t unit = by_rows ? 32 * kRowWaves : 64, tiles = ceil_div(g.sk, unit);
    const int each = !by_rows ? 2 : DP <= 32 ? 4 : DP <= 96 ? 2 : 1;
    // a step takes about 2.5 us, in which 10 MB of parts are written and read again
    const double join = 0.05 + (double)rows * g.d * 8e-7;
    const int splits = parts_for(wgs, tiles, seen_pairs(g) / ((double)unit * (double)g.sq), each, 2, join, 64);
    g.keys_per_split = ceil_div(tiles > 0 ? tiles : 1, splits) * unit;
    g.splits = (int)ceil_div(g.sk > 0 ? g.sk : 1, g.keys_per_split);
    Scratch part, planes;
    if (g.splits > 1) {
        const int64_t ml = ceil_div(2 * g.splits * rows, 4) * 4;
        if (!part.get(sizeof(float) * (size_t)(ml + g.splits * rows * g.d))) return BH_ENOMEM;
        g.part_ml = (float*)part.p;
        g.part_o = g.part_ml + ml;
    }
    int rc;
    if (by_rows) {
        hipLaunchKernelGGL(relattn_rows_kernel<DP>, dim3((unsigned)wgs, (unsigned)g.splits), dim3(64 * kRowWaves), 0, stream(), g, (int)row_tiles);
        rc = BH_LAUNCH_CHECK("bh_relbias_attention_forward");
    } else {
        g.k_blocks = (int)ceil_div(g.sk, 64) * 2;
        const size_t bytes = (size_t)g.batch * g.kv_heads * g.k_blocks * Block<DP>::BYTES;
        if (g.sk > 0) {
            if (!planes.get(2 * bytes)) return BH_ENOMEM;
            g.k_row = (const char*)planes.p;
            g.v_col = g.k_row + bytes;
            Planes p;
            p.add(g.k, g.ks, g.kv_heads, g.batch, g.sk, g.kv_len, g.k_blocks, g.vec_k, g.k_row, nullptr);
            p.add(g.v, g.vs, g.kv_heads, g.batch, g.sk, g.kv_len, g.k_blocks, g.vec_v, nullptr, g.v_col);
            rc = p.launch<DP>(g.d);
            if (rc) return rc;
        }
        rc = launch_lds(&relattn_forward_kernel<DP>, raised, dim3((unsigned)wgs, (unsigned)g.splits), ForwardLds<DP>::BYTES,
                        "bh_relbias_attention_forward", g);
    }
    if (rc || g.splits == 1) return rc;
    hipLaunchKernelGGL(relattn_join_kernel, dim3((unsigned)ceil_div(rows, 16)), dim3(256), 0, stream(), g);
    return BH_LAUNCH_CHECK("bh_relbias_attention_forward: join");
}

// The same for the backward pass, whose two walks share a launch.  A step over the queries of a key tile (four products) counts
// 4, one over the keys of a query tile (three) 3; a unit is 0.78 us at head size 64 for a workgroup that has its compute unit to
// itself, two that share one take 1.45 times as long each.  The longest walk, or all of them spread evenly and what runs last
// (three quarters of a mean walk, 0.4 where workgroups do not share a unit); parts are written and read at 4 MB in 0.72 us.  The
// constants are a fit to 13 shapes in 1 to 12 parts (within 13 %).  Us whole / in parts as chosen: 8 heads of 64 queries over 4096
// keys 298 / 61, 16 heads of 512 69 / 49, 16 heads of 2048 248 / 230; 128 heads of 1024 459 in one part, 536 in two, 96 of 128 41
// in one, 51 in four.
struct Walk { int64_t groups, longest; double mean, part_bytes; };
static void backward_parts(const Walk& keys, const Walk& queries, int each, double size, int& key_parts, int& query_parts) {
    static const int choices[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32};
    constexpr double kStart = 0.85, kBytes = 4.3e6;
    const double last = each == 2 ? 0.75 : 0.4;
    double least = INFINITY;
    for (int sk : choices)
        for (int sq : choices) {
            if ((sk > 1 && sk > keys.longest) || (sq > 1 && sq > queries.longest)) continue;
            const double a = 4 * ((double)ceil_div(keys.longest, sk) + kStart), b = 3 * ((double)ceil_div(queries.longest, sq) + kStart);
            const double am = 4 * (keys.mean / sk + kStart), bm = 3 * (queries.mean / sq + kStart);
            const double even = ((double)keys.groups * sk * am + (double)queries.groups * sq * bm) / (256.0 * each) * (each == 2 ? 1.45 : 1.0) +
                                last * (am < bm ? am : bm);
            const double walks = even > a ? (even > b ? even : b) : a > b ? a : b;
            const double parts = (sk > 1 ? keys.part_bytes * sk : 0.0) + (sq > 1 ? queries.part_bytes * sq : 0.0);
            const double cost = walks + parts / (kBytes * size);
            if (cost < 0.96 * least) { least = cost; key_parts = sk; query_parts = sq; }
        }
    if (g_force_splits > 0) {
        key_parts = (int)(g_force_splits < keys.longest ? g_force_splits : keys.longest > 0 ? keys.longest : 1);
        query_parts = (int)(g_force_splits < queries.longest ? g_force_splits : queries.longest > 0 ? queries.longest : 1);
    }
}

template <int DP>
static int run_backward(RelArgs& g, float* dtable, int accumulate) {
    static bool raised = false;
    const int64_t nbh = (int64_t)g.batch * g.heads, rows = nbh * g.sq, wgs = (int64_t)g.q_tiles * nbh;
    const int k_tiles = (int)ceil_div(g.sk, 128), each = DP <= 64 ? 2 : 1;
    // dQ walks over a tile's keys, dK and dV over the queries that see one
    const int64_t k_steps = ceil_div(g.sk, 32), q_steps = ceil_div(g.sq, 32);
    const double pairs = seen_pairs(g);
    int key_parts = 1, query_parts = 1;
    backward_parts({k_tiles * nbh, q_steps, g.sk > 0 ? pairs / (32.0 * g.sk) : 0.0, 16.0 * nbh * g.sk * g.d},
                   {wgs, k_steps, pairs / (32.0 * g.sq), 8.0 * rows * g.d}, each, DP / 64.0, key_parts, query_parts);
    g.keys_per_split = ceil_div(k_steps > 0 ? k_steps : 1, query_parts) * 32;
    g.splits = g.sk > 0 ? (int)ceil_div(g.sk, g.keys_per_split) : 1;
    g.queries_per_split = (int)ceil_div(q_steps, key_parts) * 32;
    g.q_splits = (int)ceil_div(g.sq, g.queries_per_split);
    Scratch delta, table, planes, part_q, part_kv;
    if (!delta.get(sizeof(float) * (size_t)rows) || !table.get(sizeof(double) * (size_t)g.splits * (size_t)wgs * (size_t)g.buckets)) return BH_ENOMEM;
    g.delta = (float*)delta.p;
    g.part_table = (double*)table.p;
    if (g.splits > 1) {
        if (!part_q.get(sizeof(float) * (size_t)g.splits * (size_t)rows * g.d)) return BH_ENOMEM;
        g.part_q = (float*)part_q.p;
    }
    if (g.sk > 0 && (g.group > 1 || g.q_splits > 1)) {
        const size_t size = (size_t)g.q_splits * nbh * (size_t)g.sk * g.d;
        if (!part_kv.get(2 * sizeof(float) * size)) return BH_ENOMEM;
        g.part_k = (float*)part_kv.p;
        g.part_v = g.part_k + size;
    }
    g.k_blocks = (int)ceil_div(g.sk, 64) * 2;
    g.q_blocks = (int)ceil_div(g.sq, 32);
    const size_t kb = (size_t)g.batch * g.kv_heads * g.k_blocks * Block<DP>::BYTES, qb = (size_t)nbh * g.q_blocks * Block<DP>::BYTES;
    if (!planes.get(3 * kb + 4 * qb)) return BH_ENOMEM;       // no keys: the planes of the queries alone are made, for the dots
    g.k_row = (const char*)planes.p; g.k_col = g.k_row + kb; g.v_row = g.k_col + kb;
    g.q_row = g.v_row + kb; g.q_col = g.q_row + qb; g.g_row = g.q_col + qb; g.g_col = g.g_row + qb;
    Planes p;
    if (g.sk > 0) {
        p.add(g.k, g.ks, g.kv_heads, g.batch, g.sk, g.kv_len, g.k_blocks, g.vec_k, g.k_row, g.k_col);
        p.add(g.v, g.vs, g.kv_heads, g.batch, g.sk, g.kv_len, g.k_blocks, g.vec_v, g.v_row, nullptr);
    }
    p.add(g.q, g.qs, g.heads, g.batch, g.sq, nullptr, g.q_blocks, g.vec_q, g.q_row, g.q_col);
    p.add(g.d_out, g.os, g.heads, g.batch, g.sq, nullptr, g.q_blocks, g.vec_o, g.g_row, g.g_col);
    p.last().with = g.out_in;
    p.last().dots = g.delta;
    int rc = p.launch<DP>(g.d);
    if (rc) return rc;
    constexpr int lds = KeyLds<DP>::BYTES > QueryLds<DP>::BYTES ? KeyLds<DP>::BYTES : QueryLds<DP>::BYTES;
    if (!raised) {
        rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(&relattn_backward_kernel<DP>), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
                       "bh_relbias_attention_backward: LDS size");
        if (rc) return rc;
        raised = true;
    }
    const int64_t groups = k_tiles * nbh * g.q_splits + wgs * g.splits;
    hipLaunchKernelGGL(relattn_backward_kernel<DP>, dim3((unsigned)groups), dim3(kThreads), lds, stream(), g, (int)(k_tiles * nbh), (int)wgs);
    rc = BH_LAUNCH_CHECK("bh_relbias_attention_backward");
    if (rc) return rc;
    const int per_block = g.d <= 64 ? 16 : 8;
    const auto blocks = [&](int64_t n) { const int64_t b = ceil_div(n, per_block); return (int)(b < 4096 ? b : 4096); };
    const Fold f = {(int)ceil_div(g.buckets, 16) * g.heads, g.splits > 1 ? blocks(rows) : 0,
                    g.part_k ? blocks((int64_t)g.batch * g.kv_heads * g.sk) : 0, dtable, accumulate};
    hipLaunchKernelGGL(relattn_fold_kernel, dim3((unsigned)(f.table_blocks + f.q_blocks + f.k_blocks)), dim3(256), 0, stream(), g, f);
    return BH_LAUNCH_CHECK("bh_relbias_attention_backward: fold");
}

}  // namespace bh

using namespace bh;

extern "C" {

int bh_relative_position_bucket(int64_t relative, int num_buckets, int max_distance, int bidirectional) {
    Buckets b;
    if (!make_buckets(num_buckets, max_distance, bidirectional, b)) {
        set_error(BH_EINVAL, "bh_relative_position_bucket: 2 to %d buckets (4 or more and even for both directions) and a distance past half of a direction's", kMaxBuckets);
        return BH_EINVAL;
    }
    const int first = b.both && relative > 0 ? b.side : 0;
    const uint64_t n = relative < 0 ? 0 - (uint64_t)relative : b.both ? (uint64_t)relative : 0;
    if (n < (uint64_t)b.exact) return first + (int)n;
    int f = 0;
    while (f + 1 < b.far && n >= (uint64_t)b.border[f + 1]) f++;
    return first + b.exact + f;
}

int bh_relbias_attention_force_rows(int mode) {
    BH_CHECK_ARG(mode >= -1 && mode <= 1, "-1, 0 or 1");
    g_force_rows = mode;
    return BH_OK;
}

int bh_relbias_attention_force_splits(int splits) {
    BH_CHECK_ARG(splits >= 0 && splits <= 64, "0 to 64");
    g_force_splits = splits;
    return BH_OK;
}

int bh_relbias_attention_forward(const bh_relbias_attention_t* p, const float* q, const float* k, const float* v, const float* table,
                                 const int32_t* kv_len, float* out, float* lse) {
    RelArgs g = {};
    int rc = relattn_args(__func__, p, g);
    if (rc) return rc;
    if (g.batch == 0 || g.heads == 0 || g.sq == 0) return BH_OK;
    BH_CHECK_ARG(q && out && lse && table && ((k && v) || g.sk == 0), "null pointer");
    BH_CHECK_ARG(rows_apart(g.os, g.batch, g.heads, g.sq, g.d), "output rows overlap");
    BH_REQUIRE_INIT();
    BH_CALL_GUARD();
    g.q = q; g.k = k; g.v = v; g.table = table; g.kv_len = kv_len; g.out = out; g.lse = lse;
    g.vec_q = vectors(q, g.qs, g.d); g.vec_k = vectors(k, g.ks, g.d); g.vec_v = vectors(v, g.vs, g.d); g.vec_o = vectors(out, g.os, g.d);
    ProfScope prof(BH_PROF_SDPA_FWD, 4.0 * g.batch * g.heads * (double)g.sq * (double)g.sk * g.d);
    return g.d <= 32 ? run_forward<32>(g) : g.d <= 64 ? run_forward<64>(g) : g.d <= 96 ? run_forward<96>(g) : run_forward<128>(g);
}

int bh_relbias_attention_backward(const bh_relbias_attention_t* p, const float* q, const float* k, const float* v, const float* table,
                                  const int32_t* kv_len, const float* out, const float* lse, const float* d_out, float* dq, float* dk, float* dv,
                                  float* dtable, int accumulate_table) {
    RelArgs g = {};
    int rc = relattn_args(__func__, p, g);
    if (rc) return rc;
    const bool no_queries = g.batch == 0 || g.heads == 0 || g.sq == 0;
    BH_CHECK_ARG(no_queries || (q && out && lse && d_out && dq && table && dtable && ((k && v && dk && dv) || g.sk == 0)), "null pointer");
    BH_CHECK_ARG(!no_queries || g.batch == 0 || g.heads == 0 || g.sk == 0, "keys without queries have no gradient here");
    BH_CHECK_ARG(rows_apart(g.qs, g.batch, g.heads, g.sq, g.d) && rows_apart(g.ks, g.batch, g.kv_heads, g.sk, g.d) &&
                 rows_apart(g.vs, g.batch, g.kv_heads, g.sk, g.d), "gradient rows overlap");
    if (no_queries) return BH_OK;
    BH_REQUIRE_INIT();
    BH_CALL_GUARD();
    g.q = q; g.k = k; g.v = v; g.table = table; g.kv_len = kv_len; g.out_in = out; g.lse_in = lse; g.d_out = d_out;
    g.dq = dq; g.dk = dk; g.dv = dv;
    g.vec_q = vectors(q, g.qs, g.d) && aligned16(dq); g.vec_k = vectors(k, g.ks, g.d) && aligned16(dk);
    g.vec_v = vectors(v, g.vs, g.d) && aligned16(dv); g.vec_o = vectors(d_out, g.os, g.d);
    ProfScope prof(BH_PROF_SDPA_BWD, 8.0 * g.batch * g.heads * (double)g.sq * (double)g.sk * g.d);
    return g.d <= 32 ? run_backward<32>(g, dtable, accumulate_table) : g.d <= 64 ? run_backward<64>(g, dtable, accumulate_table)
         : g.d <= 96 ? run_backward<96>(g, dtable, accumulate_table) : run_backward<128>(g, dtable, accumulate_table);
}

}  // extern "C"
