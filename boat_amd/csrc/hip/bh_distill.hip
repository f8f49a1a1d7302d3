// bh_distill.hip - distillation from a teacher's top logits, with the hard-label cross entropy mixed in.
//
// For a row of student logits z[vocab], temperature T and the teacher's kept logits t_j at vocabulary indices i_j:
//   p = softmax_j(t / T) over the kept entries,  q = softmax(z / T),  r = softmax(z)
//   row loss  l = alpha T^2 sum_j p_j (log p_j - log q_{i_j})  +  (1 - alpha) (-log r_label)
//   gradient  dl/dz = alpha T (q - p) + (1 - alpha) (r - onehot(label))
// Both softmaxes share the row's maximum, so one pass over z gives max, sum exp((z - max)/T) and sum exp(z - max), and a second
// one writes the gradient.  The kernels are bound by memory: z is read once and dz written once.  A row's workgroup keeps
// the row in registers between the two passes (up to 64 floats a thread); only what does not fit is read again, out of the
// memory-side cache.  A few long rows are cut into segments over the whole chip instead: one launch for the segments'
// statistics, one that joins them and writes the gradient.
//
// The gradient differs from the dense part at no more than topk + 1 places.  Their values are computed whole (dense part less
// the weights of every entry of that index, first entry of an index only: no atomics, the same index may come twice) and
// written over the dense ones behind a barrier.
#include "bh_common.h"

#include <math.h>

namespace bh {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // rows of odd length start anywhere

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxTopk = 4096;

struct DistillArgs {
    const float* z; int64_t ldz;
    const float* teacher; const int32_t* index;   // [rows, topk]
    const int32_t* labels;                         // [rows] or NULL
    int64_t rows; int vocab; int topk;
    float cold;                                    // log2(e) / T
    float inv_t, w_soft, w_hard;                   // 1/T, alpha T^2, 1 - alpha (0 without labels)
    float g_soft, g_hard;                          // scale alpha T, scale (1 - alpha)
    const float* seed;                             // device scalar on the gradient, or NULL
    float* row_loss; float* stats;                 // stats: [rows][3] max, sum at T, sum at 1
    float* dz; int64_t ldd;
    int segments, per_segment;                     // per_segment: a multiple of 4
    float* seg_stats; float* seg_logit;            // [rows][segments][3], [rows][topk + 1]
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// running maximum and the two sums of a part of a row
struct RowStats {
    float m, st, s1;
    __device__ __forceinline__ static float base(float m) { return m == -INFINITY ? 0.f : m; }   // a part that is all -inf
    __device__ __forceinline__ void join(const RowStats& o, float cold) {
        const float n = fmaxf(m, o.m), b = base(n);
        st = st * fast_exp2((m - b) * cold) + o.st * fast_exp2((o.m - b) * cold);
        s1 = s1 * fast_exp2((m - b) * kLog2e) + o.s1 * fast_exp2((o.m - b) * kLog2e);
        m = n;
    }
};

template <int N>
__device__ __forceinline__ void stats_of(const f32x4 (&v)[N], float cold, bool hard, RowStats& s) {
    float top = s.m;
#pragma unroll
    for (int i = 0; i < N; i++) top = fmaxf(fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3])), top);
    const float b = RowStats::base(top);
    float a = s.st * fast_exp2((s.m - b) * cold), c = s.s1 * fast_exp2((s.m - b) * kLog2e);
#pragma unroll
    for (int i = 0; i < N; i++) {
#pragma unroll
        for (int q = 0; q < 4; q++) a += fast_exp2((v[i][q] - b) * cold);
        __builtin_amdgcn_sched_barrier(0);   // one vector's temporaries at a time: the registers hold the row
    }
    if (hard) {
        float again = b;                     // ... and the differences are taken anew
        asm volatile("" : "+v"(again));
#pragma unroll
        for (int i = 0; i < N; i++) {
#pragma unroll
            for (int q = 0; q < 4; q++) c += fast_exp2((v[i][q] - again) * kLog2e);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    s.m = top; s.st = a; s.s1 = c;
}

template <int NWAVES>
__device__ __forceinline__ RowStats block_stats(RowStats s, float cold, float (*red)[3]) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const RowStats o = {__shfl_xor(s.m, off, 64), __shfl_xor(s.st, off, 64), __shfl_xor(s.s1, off, 64)};
        s.join(o, cold);
    }
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (lane == 0) { red[w][0] = s.m; red[w][1] = s.st; red[w][2] = s.s1; }
    __syncthreads();
    RowStats t = {red[0][0], red[0][1], red[0][2]};
#pragma unroll
    for (int i = 1; i < NWAVES; i++) t.join(RowStats{red[i][0], red[i][1], red[i][2]}, cold);
    return t;
}

// A part [begin, end) of a row: vectors of four from begin on, and up to three elements behind them, one to a thread.
// Loads past the last vector read the last one and count as -inf, so that no branch stands between a thread's loads.
struct Span {
    const float* z;
    int vecs, tail;            // whole vectors; elements behind them
    __device__ __forceinline__ Span(const float* row, int begin, int end) : z(row + begin), vecs((end - begin) >> 2), tail((end - begin) & 3) {}
    __device__ __forceinline__ f32x4 load(int i) const {
        f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (vecs > 0) {        // the same for the whole launch
            const f32x4 u = *reinterpret_cast<const f32x4u*>(z + 4 * (unsigned)min(i, vecs - 1));
            if (i < vecs) v = u;
        }
        return v;
    }
    __device__ __forceinline__ float rest(int tid) const { return tid < tail ? z[4 * vecs + tid] : -INFINITY; }
};
__device__ __forceinline__ void stats_of_one(float x, float cold, RowStats& s) {
    s.join(RowStats{x, x == -INFINITY ? 0.f : 1.f, x == -INFINITY ? 0.f : 1.f}, cold);
}

// ---- the special places of a row: the teacher's entries and, last, the label, staged in LDS
struct Entries {
    int* index;       // [topk + 1], -1 = left out
    float* value;     // [topk + 1] teacher logit / T
    float* logit;     // [topk + 1] student logit at the index
};
__device__ __forceinline__ Entries entries_at(float* lds, int n) { return {reinterpret_cast<int*>(lds), lds + n, lds + 2 * n}; }

__device__ __forceinline__ void stage_entries(const DistillArgs& g, int64_t row, const Entries& e, const float* z, const float* gathered,
                                              int threads) {
    for (int j = threadIdx.x; j <= g.topk; j += threads) {
        int i = -1;
        float t = -INFINITY, x = 0.f;
        if (j < g.topk) {
            i = g.index[row * g.topk + j];
            t = g.teacher[row * g.topk + j] * g.inv_t;
        } else if (g.labels) {
            i = g.labels[row];
        }
        if (i < 0 || i >= g.vocab) i = -1;
        if (i < 0) t = -INFINITY; else x = gathered ? gathered[row * (g.topk + 1) + j] : z[i];
        e.index[j] = i;
        e.value[j] = t;
        e.logit[j] = x;
    }
}
// maximum and sum of the teacher's softmax, by every wavefront on its own
__device__ __forceinline__ void teacher_softmax(const DistillArgs& g, const Entries& e, float& top, float& inv_sum) {
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    for (int j = lane; j < g.topk; j += 64) m = fmaxf(m, e.value[j]);
    m = wave_max(m);
    float s = 0.f;
    if (m > -INFINITY)
        for (int j = lane; j < g.topk; j += 64) s += fast_exp2((e.value[j] - m) * kLog2e);
    s = wave_sum(s);
    top = m;
    inv_sum = s;   // the sum itself: 0 when nothing is kept
}

// the row's loss, by one wavefront
__device__ __forceinline__ float row_loss_of(const DistillArgs& g, const Entries& e, const RowStats& s, float top, float sum) {
    const int lane = threadIdx.x & 63;
    const float b = RowStats::base(s.m);
    float acc = 0.f;
    if (sum != 0.f) {
        const float ls = logf(sum), lt = logf(s.st), inv = 1.f / sum;
        for (int j = lane; j < g.topk; j += 64) {
            const float lp = e.value[j] - top, p = fast_exp2(lp * kLog2e) * inv;
            if (p > 0.f || p != p) acc += p * ((lp - ls) - ((e.logit[j] - b) * g.inv_t - lt));
        }
    }
    acc = wave_sum(acc) * g.w_soft;
    if (g.w_hard != 0.f && e.index[g.topk] >= 0) acc += g.w_hard * (logf(s.s1) - (e.logit[g.topk] - b));
    return acc;
}

struct GradRow { float base, cold, ct, c1; };   // dz = ct exp2((z - base) cold) + c1 exp2((z - base) log2 e)

__device__ __forceinline__ GradRow grad_row(const DistillArgs& g, const Entries& e, const RowStats& s, float sum) {
    const float seed = g.seed ? g.seed[0] : 1.f;
    return {RowStats::base(s.m), g.cold, sum != 0.f ? g.g_soft * seed / s.st : 0.f,
            g.w_hard != 0.f && e.index[g.topk] >= 0 ? g.g_hard * seed / s.s1 : 0.f};
}
__device__ __forceinline__ float grad_at(const GradRow& r, float z) {
    float d = r.ct == 0.f ? 0.f : r.ct * fast_exp2((z - r.base) * r.cold);
    if (r.c1 != 0.f) d += r.c1 * fast_exp2((z - r.base) * kLog2e);
    return d;
}
__device__ __forceinline__ void grad_store(const GradRow& r, f32x4 v, float* __restrict__ dz, int i, int vecs) {
    f32x4 d;
#pragma unroll
    for (int q = 0; q < 4; q++) d[q] = grad_at(r, v[q]);
    if (i < vecs) *reinterpret_cast<f32x4u*>(dz + 4 * (unsigned)i) = d;
}
// the places of [begin, end) that the teacher or the label names, behind the dense stores
__device__ __forceinline__ void grad_entries(const DistillArgs& g, const Entries& e, const GradRow& r, float top, float sum, float* dz,
                                             int begin, int end, int threads) {
    const float seed = g.seed ? g.seed[0] : 1.f;
    const float soft = sum != 0.f ? g.g_soft * seed / sum : 0.f, hard = g.w_hard != 0.f ? g.g_hard * seed : 0.f;
    for (int j = threadIdx.x; j <= g.topk; j += threads) {
        const int i = e.index[j];
        if (i < begin || i >= end) continue;
        bool first = true;
        float w = 0.f;
        for (int o = 0; o <= g.topk; o++) {
            if (e.index[o] != i) continue;
            if (o < j) { first = false; break; }
            w += o == g.topk ? hard : soft == 0.f ? 0.f : soft * fast_exp2((e.value[o] - top) * kLog2e);
        }
        if (first) dz[i] = grad_at(r, e.logit[j]) - w;
    }
}

// ---- one workgroup per row: statistics, loss and (GRAD) gradient; NV * 4 floats a thread stay in registers between the two
template <int THREADS, int NV, bool GRAD>
__global__ __launch_bounds__(THREADS) void distill_row_kernel(DistillArgs g) {
    extern __shared__ float lds[];
    __shared__ float red[THREADS / 64][3];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const Span part(g.z + row * g.ldz, 0, g.vocab);
    const bool hard = g.w_hard != 0.f;
    f32x4 v[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) v[i] = part.load(tid + i * THREADS);
    const float rest = part.rest(tid);
    const Entries e = entries_at(lds, g.topk + 1);
    stage_entries(g, row, e, part.z, nullptr, THREADS);
    RowStats s = {-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; i += 4) {
        f32x4 u[4 < NV ? 4 : NV];
#pragma unroll
        for (int q = 0; q < (4 < NV ? 4 : NV); q++) u[q] = v[i + q];
        stats_of(u, g.cold, hard, s);
        __builtin_amdgcn_sched_barrier(0);
    }
    for (int at = NV * THREADS + tid; at < part.vecs; at += 4 * THREADS) {
        f32x4 u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = part.load(at + i * THREADS);
        stats_of(u, g.cold, hard, s);
    }
    if (tid < part.tail) stats_of_one(rest, g.cold, s);
    s = block_stats<THREADS / 64>(s, g.cold, red);       // its barrier also publishes the entries
    float top, sum;
    teacher_softmax(g, e, top, sum);
    if (tid < 64) {
        const float l = row_loss_of(g, e, s, top, sum);
        if (tid == 0) {
            g.row_loss[row] = l;
            if (g.stats) { g.stats[3 * row] = s.m; g.stats[3 * row + 1] = s.st; g.stats[3 * row + 2] = s.s1; }
        }
    }
    if (!GRAD) return;
    float* dz = g.dz + row * g.ldd;
    const GradRow r = grad_row(g, e, s, sum);
    int again = tid;                                     // the stores' offsets are computed anew, not kept since the loads
    asm volatile("" : "+v"(again));
#pragma unroll
    for (int i = 0; i < NV; i++) {
        grad_store(r, v[i], dz, again + i * THREADS, part.vecs);
        __builtin_amdgcn_sched_barrier(0);               // four gradients in registers at a time, not all
    }
    for (int at = NV * THREADS + tid; at < part.vecs; at += 4 * THREADS) {
        f32x4 u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = part.load(at + i * THREADS);
#pragma unroll
        for (int i = 0; i < 4; i++) grad_store(r, u[i], dz, at + i * THREADS, part.vecs);
    }
    if (tid < part.tail) dz[4 * part.vecs + tid] = grad_at(r, rest);
    __syncthreads();
    grad_entries(g, e, r, top, sum, dz, 0, g.vocab, THREADS);
}

// ---- rows cut into segments
constexpr int kSegThreads = 256;
__global__ __launch_bounds__(kSegThreads) void distill_segment_stats_kernel(DistillArgs g) {
    __shared__ float red[kSegThreads / 64][3];
    const int64_t row = blockIdx.y;
    const int begin = blockIdx.x * g.per_segment, end = min(g.vocab, begin + g.per_segment);
    const float* z = g.z + row * g.ldz;
    // logits at the named places: the gradient may be written over z before another segment's workgroup looks for them
    for (int j = threadIdx.x; j <= g.topk; j += kSegThreads) {
        const int i = j < g.topk ? g.index[row * g.topk + j] : g.labels ? g.labels[row] : -1;
        if (i >= begin && i < end) g.seg_logit[row * (g.topk + 1) + j] = z[i];
    }
    RowStats s = {-INFINITY, 0.f, 0.f};
    const Span part(z, begin, end);
    for (int at = threadIdx.x; at < part.vecs; at += 4 * kSegThreads) {
        f32x4 u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = part.load(at + i * kSegThreads);
        stats_of(u, g.cold, g.w_hard != 0.f, s);
    }
    if ((int)threadIdx.x < part.tail) stats_of_one(part.rest(threadIdx.x), g.cold, s);
    s = block_stats<kSegThreads / 64>(s, g.cold, red);
    if (threadIdx.x == 0) {
        float* o = g.seg_stats + 3 * (row * g.segments + blockIdx.x);
        o[0] = s.m; o[1] = s.st; o[2] = s.s1;
    }
}

// joins the segments' statistics (by every wavefront: a lane per segment)
__device__ __forceinline__ RowStats joined_stats(const DistillArgs& g, int64_t row) {
    RowStats s = {-INFINITY, 0.f, 0.f};
    for (int i = threadIdx.x & 63; i < g.segments; i += 64) {
        const float* o = g.seg_stats + 3 * (row * g.segments + i);
        s.join(RowStats{o[0], o[1], o[2]}, g.cold);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const RowStats o = {__shfl_xor(s.m, off, 64), __shfl_xor(s.st, off, 64), __shfl_xor(s.s1, off, 64)};
        s.join(o, g.cold);
    }
    return s;
}

// the gradient of a row's segment from statistics: the segments' (with the row's loss), or those a forward call kept
template <bool JOIN, bool GRAD>
__global__ __launch_bounds__(kSegThreads) void distill_segment_grad_kernel(DistillArgs g) {
    extern __shared__ float lds[];
    const int64_t row = blockIdx.y;
    const int begin = GRAD ? blockIdx.x * g.per_segment : 0, end = GRAD ? min(g.vocab, begin + g.per_segment) : 0;
    const float* z = g.z + row * g.ldz;
    const Entries e = entries_at(lds, g.topk + 1);
    if (JOIN) {
        stage_entries(g, row, e, z, g.seg_logit, kSegThreads);
    } else {
        // only this segment's logits: others' may be overwritten already
        for (int j = threadIdx.x; j <= g.topk; j += kSegThreads) {
            int i = j < g.topk ? g.index[row * g.topk + j] : g.labels ? g.labels[row] : -1;
            if (i < 0 || i >= g.vocab) i = -1;
            e.index[j] = i;
            e.value[j] = j < g.topk && i >= 0 ? g.teacher[row * g.topk + j] * g.inv_t : -INFINITY;
            e.logit[j] = i >= begin && i < end ? z[i] : 0.f;
        }
    }
    RowStats s;
    if (JOIN) s = joined_stats(g, row);
    else s = RowStats{g.stats[3 * row], g.stats[3 * row + 1], g.stats[3 * row + 2]};
    __syncthreads();
    float top, sum;
    teacher_softmax(g, e, top, sum);
    if (JOIN && blockIdx.x == 0 && threadIdx.x < 64) {
        const float l = row_loss_of(g, e, s, top, sum);
        if (threadIdx.x == 0) {
            g.row_loss[row] = l;
            if (g.stats) { g.stats[3 * row] = s.m; g.stats[3 * row + 1] = s.st; g.stats[3 * row + 2] = s.s1; }
        }
    }
    if (!GRAD) return;
    float* dz = g.dz + row * g.ldd;
    const GradRow r = grad_row(g, e, s, sum);
    const Span part(z, begin, end);
    for (int at = threadIdx.x; at < part.vecs; at += 4 * kSegThreads) {
        f32x4 u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = part.load(at + i * kSegThreads);
#pragma unroll
        for (int i = 0; i < 4; i++) grad_store(r, u[i], dz + begin, at + i * kSegThreads, part.vecs);
    }
    if ((int)threadIdx.x < part.tail) dz[begin + 4 * part.vecs + threadIdx.x] = grad_at(r, part.rest(threadIdx.x));
    __syncthreads();
    grad_entries(g, e, r, top, sum, dz, begin, end, kSegThreads);
}

// loss = scale * sum of the rows' losses, in a fixed order
__global__ __launch_bounds__(1024) void distill_loss_kernel(const float* __restrict__ row_loss, int64_t rows, float scale, float* out) {
    __shared__ double red[16];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += 1024) s += (double)row_loss[i];
    s = wave_sum_f64(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 16; i++) t += red[i];
        out[0] = (float)(t * (double)scale);
    }
}

static int distill_check(const char* fn, const float* z, int64_t ldz, const float* teacher, const int32_t* index, int64_t rows, int64_t vocab,
                         int64_t topk, float temperature, float alpha) {
    if (rows < 0 || vocab < 1 || topk < 0) return set_error(BH_EINVAL, "%s: rows >= 0, vocab >= 1 and topk >= 0 are needed", fn);
    if (vocab > (1 << 30) || rows > 65535 * (int64_t)32768) return set_error(BH_EINVAL, "%s: too many rows or too large a vocabulary", fn);
    if (topk > kMaxTopk) return set_error(BH_EINVAL, "%s: topk is at most %d", fn, kMaxTopk);
    if (ldz < vocab) return set_error(BH_EINVAL, "%s: leading dimension too small", fn);
    if (!(temperature > 0.f) || !(temperature < INFINITY)) return set_error(BH_EINVAL, "%s: the temperature is a positive number", fn);
    if (!(alpha >= 0.f && alpha <= 1.f)) return set_error(BH_EINVAL, "%s: alpha lies in [0, 1]", fn);
    if (rows > 0 && (!z || (topk > 0 && (!teacher || !index)))) return set_error(BH_EINVAL, "%s: null pointer", fn);
    return BH_OK;
}

static DistillArgs distill_args(const float* z, int64_t ldz, const float* teacher, const int32_t* index, const int32_t* labels, int64_t rows,
                                int64_t vocab, int64_t topk, float temperature, float alpha, float scale) {
    DistillArgs g = {};
    g.z = z; g.ldz = ldz; g.teacher = teacher; g.index = index; g.labels = labels;
    g.rows = rows; g.vocab = (int)vocab; g.topk = (int)topk;
    g.inv_t = 1.f / temperature;
    g.cold = kLog2e / temperature;
    g.w_soft = alpha * temperature * temperature;
    g.w_hard = labels ? 1.f - alpha : 0.f;
    g.g_soft = scale * alpha * temperature;
    g.g_hard = scale * (1.f - alpha);
    return g;
}

// segments of a row so that a few rows still fill the chip; 1 = a workgroup per row
static int segments_for(int64_t rows, int64_t vocab) {
    if (rows >= 256 || vocab < 8192) return 1;
    const int64_t want = ceil_div(512, rows), most = ceil_div(vocab, 4096);
    return (int)(want < most ? want : most);
}
static void cut_row(DistillArgs& g, int segments) {
    g.per_segment = (int)(ceil_div(ceil_div(g.vocab, segments), 4) * 4);
    g.segments = (int)ceil_div(g.vocab, g.per_segment);
}

template <bool GRAD>
static int launch_rows(const DistillArgs& g) {
    const size_t lds = sizeof(float) * 3 * (size_t)(g.topk + 1);
    const dim3 grid((unsigned)g.rows);
    // the gradient's rows stay in registers (as many threads as it takes, up to the 64 K floats of a compute unit); without
    // one the row only streams through
    if (!GRAD && g.vocab > 4096) hipLaunchKernelGGL((distill_row_kernel<512, 8, GRAD>), grid, dim3(512), lds, stream(), g);
    else if (g.vocab <= 1024) hipLaunchKernelGGL((distill_row_kernel<256, 1, GRAD>), grid, dim3(256), lds, stream(), g);
    else if (g.vocab <= 4096) hipLaunchKernelGGL((distill_row_kernel<256, 4, GRAD>), grid, dim3(256), lds, stream(), g);
    else if (g.vocab <= 16384) hipLaunchKernelGGL((distill_row_kernel<256, 16, GRAD>), grid, dim3(256), lds, stream(), g);
    else if (g.vocab <= 32768) hipLaunchKernelGGL((distill_row_kernel<512, 16, GRAD>), grid, dim3(512), lds, stream(), g);
    else hipLaunchKernelGGL((distill_row_kernel<1024, 16, GRAD>), grid, dim3(1024), lds, stream(), g);
    return BH_LAUNCH_CHECK("bh_distill");
}

template <bool GRAD>
static int run_distill(DistillArgs g, float scale, float* loss_out) {
    Scratch own_rows, seg;
    if (!g.row_loss) {
        if (!own_rows.get(sizeof(float) * (size_t)g.rows)) return BH_ENOMEM;
        g.row_loss = (float*)own_rows.p;
    }
    const int segments = segments_for(g.rows, g.vocab);
    int rc;
    if (segments == 1) {
        rc = launch_rows<GRAD>(g);
    } else {
        cut_row(g, segments);
        const size_t words = (size_t)g.rows * (3 * (size_t)g.segments + (size_t)g.topk + 1);
        if (!seg.get(sizeof(float) * words)) return BH_ENOMEM;
        g.seg_stats = (float*)seg.p;
        g.seg_logit = g.seg_stats + 3 * (size_t)g.rows * (size_t)g.segments;
        hipLaunchKernelGGL(distill_segment_stats_kernel, dim3((unsigned)g.segments, (unsigned)g.rows), dim3(kSegThreads), 0, stream(), g);
        rc = BH_LAUNCH_CHECK("bh_distill: segments");
        if (rc) return rc;
        const size_t lds = sizeof(float) * 3 * (size_t)(g.topk + 1);
        hipLaunchKernelGGL((distill_segment_grad_kernel<true, GRAD>), dim3(GRAD ? (unsigned)g.segments : 1u, (unsigned)g.rows),
                           dim3(kSegThreads), lds, stream(), g);
        rc = BH_LAUNCH_CHECK("bh_distill: join");
    }
    if (rc || !loss_out) return rc;
    hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(1024), 0, stream(), (const float*)g.row_loss, g.rows, scale, loss_out);
    return BH_LAUNCH_CHECK("bh_distill: loss");
}

}  // namespace bh

using namespace bh;

extern "C" {

int bh_distill_forward(const float* logits, int64_t ld, const float* teacher, const int32_t* index, const int32_t* labels, int64_t rows,
                       int64_t vocab, int64_t topk, float temperature, float alpha, float scale, float* row_loss, float* stats, float* loss_out) {
    int rc = distill_check(__func__, logits, ld, teacher, index, rows, vocab, topk, temperature, alpha);
    if (rc) return rc;
    BH_REQUIRE_INIT();
    BH_CALL_GUARD();
    if (rows == 0) return loss_out ? bh_fill(loss_out, 0.f, 1) : BH_OK;
    DistillArgs g = distill_args(logits, ld, teacher, index, labels, rows, vocab, topk, temperature, alpha, scale);
    g.row_loss = row_loss; g.stats = stats;
    return run_distill<false>(g, scale, loss_out);
}

int bh_distill_backward(const float* logits, int64_t ld, const float* teacher, const int32_t* index, const int32_t* labels, int64_t rows,
                        int64_t vocab, int64_t topk, float temperature, float alpha, float scale, const float* stats, const float* seed,
                        float* dlogits, int64_t ldd) {
    int rc = distill_check(__func__, logits, ld, teacher, index, rows, vocab, topk, temperature, alpha);
    if (rc) return rc;
    BH_CHECK_ARG(ldd >= vocab, "leading dimension too small");
    BH_CHECK_ARG(dlogits != logits || ldd == ld, "a gradient in place has the logits' leading dimension");
    BH_CHECK_ARG((stats && dlogits) || rows == 0, "null pointer");
    BH_REQUIRE_INIT();
    BH_CALL_GUARD();
    if (rows == 0) return BH_OK;
    DistillArgs g = distill_args(logits, ld, teacher, index, labels, rows, vocab, topk, temperature, alpha, scale);
    g.stats = const_cast<float*>(stats); g.seed = seed; g.dz = dlogits; g.ldd = ldd;
    // a workgroup streams a segment of at most 16 K logits; the grid's second dimension holds 65535 rows
    const int64_t by_size = ceil_div(vocab, 16384), by_rows = segments_for(rows, vocab);
    cut_row(g, (int)(by_size > by_rows ? by_size : by_rows));
    const size_t lds = sizeof(float) * 3 * (size_t)(topk + 1);
    for (int64_t r0 = 0; r0 < rows; r0 += 65535) {
        DistillArgs h = g;
        h.rows = rows - r0 < 65535 ? rows - r0 : 65535;
        h.z += r0 * ld; h.teacher += r0 * topk; h.index += r0 * topk; h.stats += 3 * r0; h.dz += r0 * ldd;
        if (h.labels) h.labels += r0;
        hipLaunchKernelGGL((distill_segment_grad_kernel<false, true>), dim3((unsigned)h.segments, (unsigned)h.rows), dim3(kSegThreads), lds,
                           stream(), h);
        rc = BH_LAUNCH_CHECK("bh_distill_backward");
        if (rc) return rc;
    }
    return BH_OK;
}

int bh_distill_loss_grad(const float* logits, int64_t ld, const float* teacher, const int32_t* index, const int32_t* labels, int64_t rows,
                         int64_t vocab, int64_t topk, float temperature, float alpha, float scale, float* row_loss, float* loss_out,
                         float* dlogits, int64_t ldd) {
    int rc = distill_check(__func__, logits, ld, teacher, index, rows, vocab, topk, temperature, alpha);
    if (rc) return rc;
    BH_CHECK_ARG(ldd >= vocab, "leading dimension too small");
    BH_CHECK_ARG(dlogits != logits || ldd == ld, "a gradient in place has the logits' leading dimension");
    BH_CHECK_ARG(dlogits || rows == 0, "null pointer");
    BH_REQUIRE_INIT();
    BH_CALL_GUARD();
    if (rows == 0) return loss_out ? bh_fill(loss_out, 0.f, 1) : BH_OK;
    DistillArgs g = distill_args(logits, ld, teacher, index, labels, rows, vocab, topk, temperature, alpha, scale);
    g.row_loss = row_loss; g.dz = dlogits; g.ldd = ldd;
    return run_distill<true>(g, scale, loss_out);
}

}  // extern "C"
