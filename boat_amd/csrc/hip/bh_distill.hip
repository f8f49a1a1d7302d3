// bh_distill.hip - distillation from a teacher's top logits, with the hard-label cross entropy mixed in.
//
// For a row of student logits z[vocab], temperature T and the teacher's kept logits t_j at vocabulary indices i_j:
//   p = softmax_j(t / T) over the kept entries,  q = softmax(z / T),  r = softmax(z)
//   row loss  l = alpha T^2 sum_j p_j (log p_j - log q_{i_j})  +  (1 - alpha) (-log r_label)
//   gradient  dl/dz = alpha T (q - p) + (1 - alpha) (r - onehot(label))
// Both softmaxes share the row's maximum, so one pass over z gives max, sum exp((z - max)/T) and sum exp(z - max), and a second
// one writes the gradient.  The kernels are bound by memory: z is read once and dz written once.  A row's workgroup keeps
// the row in registers and LDS between the two passes; only what does not fit is read again, out of the memory-side cache.
// Loss and gradient of 8192 x 50001 logits 668 us (3.28 GB, 4.9 TB/s; a large copy reaches 5.2), the loss alone of 4096 x 32000
// 88 us (5.9 TB/s).  A few long rows are cut into segments over the whole chip instead: one launch for the segments'
// statistics, one that joins them and writes the gradient.
//
// The gradient differs from the dense part at no more than topk + 1 places.  Their values are computed whole (dense part less
// the weights of every entry of that index, first entry of an index only: no atomics, the same index may come twice) and
// written over the dense ones behind a barrier.
#include "bh_common.h"

#include <float.h>
#include <math.h>

#include <type_traits>

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
    int terms;                                     // which softmaxes a row needs: kSoft, kSame or kBoth
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

// The exponents are (z - max) log2(e)/T, the maximum taken off first: their error is two roundings of themselves, however far
// the logits lie from zero, and a maximum's own exponent is 0.  (As fma(z, log2(e)/T, -max log2(e)/T) it would be the rounding of
// the second product, which differs from thread to thread with the maximum and overflows under masks like -1e10.)  The softmax at 1
// has exponentials of its own.  (Powers of the ones at T, for whole T, multiply their error by T and save next to
// nothing: 4096 x 50001 at T = 3 337 us with them, 336 without, 37 x 128001 at T = 2 17.0 and 17.4.)
enum { kSoft, kSame, kBoth };   // the softmax at T alone (no labels, or no weight on them); T = 1: both are one; two softmaxes
template <int TERMS>
__device__ __forceinline__ float hard_term(float soft, float below) {
    return TERMS == kSame ? soft : fast_exp2(below * kLog2e);
}
template <int TERMS, int N>
__device__ __forceinline__ void add_terms(const f32x4 (&v)[N], float b, float cold, float& a, float& c) {
#pragma unroll
    for (int i = 0; i < N; i++) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float below = v[i][q] - b, t = fast_exp2(below * cold);
            a += t;
            if (TERMS != kSoft) c += hard_term<TERMS>(t, below);
        }
        __builtin_amdgcn_sched_barrier(0);   // one vector's temporaries at a time: the registers hold the row
    }
}
template <int N>
__device__ __forceinline__ void stats_of(const f32x4 (&v)[N], float cold, int terms, RowStats& s) {
    float top = s.m;
#pragma unroll
    for (int i = 0; i < N; i++) top = fmaxf(fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3])), top);
    const float b = RowStats::base(top);
    float a = s.st * fast_exp2((s.m - b) * cold), c = s.s1 * fast_exp2((s.m - b) * kLog2e);
    if (terms == kSoft) add_terms<kSoft>(v, b, cold, a, c);
    else if (terms == kSame) add_terms<kSame>(v, b, cold, a, c);
    else add_terms<kBoth>(v, b, cold, a, c);
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

// A part [begin, end) of a row: up to three elements, vectors of four from the first 16-byte boundary on, up to three elements
// behind them (rows of odd length start anywhere; vectors across the boundaries cost 10 %).  The single elements are one to a
// thread.  Loads past the last vector read the last one and count as -inf, so that no branch stands between a thread's loads.
struct Span {
    const float* z;
    int head, vecs, tail;      // elements before the vectors; whole vectors; elements behind
    __device__ __forceinline__ Span(const float* row, int begin, int end) {
        const int n = end - begin;
        head = min((int)((16 - (reinterpret_cast<uintptr_t>(row + begin) & 15)) & 15) >> 2, n);
        vecs = (n - head) >> 2;
        tail = (n - head) & 3;
        z = row + begin + head;
    }
    template <bool ONCE = false>   // ONCE: not read again, does not stay in the caches
    __device__ __forceinline__ f32x4 load(int i) const {
        f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (vecs > 0) {        // the same for the whole launch
            const f32x4u* p = reinterpret_cast<const f32x4u*>(z + 4 * (unsigned)min(i, vecs - 1));
            const f32x4 u = ONCE ? __builtin_nontemporal_load(p) : *p;
            if (i < vecs) v = u;
        }
        return v;
    }
    __device__ __forceinline__ bool single(int tid) const { return tid < head + tail; }
    __device__ __forceinline__ int place(int tid) const { return tid < head ? tid - head : 4 * vecs + tid - head; }   // from z
    __device__ __forceinline__ float rest(int tid) const { return single(tid) ? z[place(tid)] : -INFINITY; }
};
__device__ __forceinline__ void stats_of_one(float x, float cold, RowStats& s) {
    s.join(RowStats{x, x == -INFINITY ? 0.f : 1.f, x == -INFINITY ? 0.f : 1.f}, cold);
}

// ---- the special places of a row: the teacher's entries and, last, the label, staged in LDS
struct Entries {
    int* index;       // [topk + 1], -1 = left out
    float* value;     // [topk + 1] teacher logit
    float* logit;     // [topk + 1] student logit at the index
};
// the indices come first and fill whole vectors of four (-2 behind the label)
__host__ __device__ __forceinline__ int entry_slots(int topk) { return (topk + 1 + 3) / 4 * 4; }
__device__ __forceinline__ Entries entries_at(float* lds, int slots) { return {reinterpret_cast<int*>(lds), lds + slots, lds + 2 * slots}; }

// entry j of a row as memory has it
struct Entry {
    int index;
    float value;
    __device__ __forceinline__ Entry(const DistillArgs& g, int64_t row, int j) : index(j > g.topk ? -2 : -1), value(-INFINITY) {
        if (j < g.topk) {
            index = g.index[row * g.topk + j];
            value = g.teacher[row * g.topk + j];
        } else if (j == g.topk && g.labels) {
            index = g.labels[row];
        }
    }
    // z: the row's logits; only those in [begin, end) are looked at
    __device__ __forceinline__ void stage(const DistillArgs& g, const Entries& e, int j, const float* z, int begin, int end) {
        if (j <= g.topk && (index < 0 || index >= g.vocab)) index = -1;
        e.index[j] = index;
        e.value[j] = index < 0 ? -INFINITY : value;
        e.logit[j] = index >= begin && index < end ? z[index] : 0.f;
    }
};
// maximum and sum of the teacher's softmax, by every wavefront on its own
__device__ __forceinline__ void teacher_softmax(const DistillArgs& g, const Entries& e, float& top, float& inv_sum) {
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    for (int j = lane; j < g.topk; j += 64) m = fmaxf(m, e.value[j]);
    m = wave_max(m);
    float s = 0.f;
    if (m > -INFINITY)
        for (int j = lane; j < g.topk; j += 64) s += fast_exp2((e.value[j] - m) * g.cold);
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
            const float below = e.value[j] - top, p = fast_exp2(below * g.cold) * inv;
            if (p > 0.f || p != p) acc += p * ((below * g.inv_t - ls) - ((e.logit[j] - b) * g.inv_t - lt));
        }
    }
    acc = wave_sum(acc) * g.w_soft;
    if (g.w_hard != 0.f && e.index[g.topk] >= 0) acc += g.w_hard * (logf(s.s1) - (e.logit[g.topk] - b));
    return acc;
}

// a row's loss and statistics, by its first wavefront
__device__ __forceinline__ void finish_row(const DistillArgs& g, const Entries& e, const RowStats& s, float top, float sum, int64_t row) {
    const float l = row_loss_of(g, e, s, top, sum);
    if (threadIdx.x == 0) {
        g.row_loss[row] = l;
        if (g.stats) { g.stats[3 * row] = s.m; g.stats[3 * row + 1] = s.st; g.stats[3 * row + 2] = s.s1; }
    }
}
// loss = scale * sum of the rows' losses, in a fixed order.  (A count of finished rows, whose last one adds them up in the same
// launch, costs more than this launch: 96 rows of 1000 logits 9.8 us against 9.2, 1024 rows 32 against 10.5.)
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

struct GradRow { float cold, base, ct, c1; int terms; };   // dz = ct exp2((z - base) cold) + c1 exp2((z - base) log2 e)

__device__ __forceinline__ GradRow grad_row(const DistillArgs& g, const Entries& e, const RowStats& s, float sum) {
    const float seed = g.seed ? g.seed[0] : 1.f, b = RowStats::base(s.m);
    const bool hard = g.w_hard != 0.f && e.index[g.topk] >= 0;
    return {g.cold, b, sum != 0.f ? g.g_soft * seed / s.st : 0.f, hard ? g.g_hard * seed / s.s1 : 0.f, g.terms};
}
template <int TERMS>
__device__ __forceinline__ float grad_term(const GradRow& r, float z) {
    const float below = z - r.base, t = fast_exp2(below * r.cold), d = r.ct * t;
    return TERMS == kSoft ? d : fmaf(r.c1, hard_term<TERMS>(t, below), d);
}
// calls f with the terms as a constant: which they are holds for the whole launch, so the choice stands outside the loops
template <typename F>
__device__ __forceinline__ void with_terms(int terms, F f) {
    if (terms == kSoft) f(std::integral_constant<int, kSoft>{});
    else if (terms == kSame) f(std::integral_constant<int, kSame>{});
    else f(std::integral_constant<int, kBoth>{});
}
__device__ __forceinline__ float grad_at(const GradRow& r, float z) {
    float d = 0.f;
    with_terms(r.terms, [&](auto t) { d = grad_term<decltype(t)::value>(r, z); });
    return d;
}
// the gradient is not read again here: its stores pass the caches by, which keep the logits (131072 logits: 476 us against 571)
template <int TERMS>
__device__ __forceinline__ void grad_store(const GradRow& r, f32x4 v, float* __restrict__ dz, int i, int vecs) {
    f32x4 d;
#pragma unroll
    for (int q = 0; q < 4; q++) d[q] = grad_term<TERMS>(r, v[q]);
    if (i < vecs) __builtin_nontemporal_store(d, reinterpret_cast<f32x4u*>(dz + 4 * (unsigned)i));
}
// the places of [begin, end) that the teacher or the label names, behind the dense stores
__device__ __forceinline__ void grad_entries(const DistillArgs& g, const Entries& e, const GradRow& r, float top, float sum, float* dz,
                                             int begin, int end, int threads) {
    const float seed = g.seed ? g.seed[0] : 1.f;
    const float soft = sum != 0.f ? g.g_soft * seed / sum : 0.f, hard = g.w_hard != 0.f ? g.g_hard * seed : 0.f;
    for (int j = threadIdx.x; j <= g.topk; j += threads) {
        const int i = e.index[j];
        if (i < begin || i >= end) continue;
        // how often does the index occur?  Mostly once; else the first entry takes the weights of all of them
        int same = 0;
        const int4* all = reinterpret_cast<const int4*>(e.index);
#pragma unroll 4
        for (int o = 0; o < entry_slots(g.topk) / 4; o++) {
            const int4 x = all[o];
            same += (x.x == i) + (x.y == i) + (x.z == i) + (x.w == i);
        }
        bool first = true;
        float w = j == g.topk ? hard : soft == 0.f ? 0.f : soft * fast_exp2((e.value[j] - top) * g.cold);
        if (same > 1) {
            w = 0.f;
            for (int o = 0; o <= g.topk; o++) {
                if (e.index[o] != i) continue;
                if (o < j) { first = false; break; }
                w += o == g.topk ? hard : soft == 0.f ? 0.f : soft * fast_exp2((e.value[o] - top) * g.cold);
            }
        }
        if (first) dz[i] = grad_at(r, e.logit[j]) - w;
    }
}

// ---- one workgroup per row: statistics, loss and (GRAD) gradient.  Between the two a thread keeps NV vectors in registers and LV
// in LDS; what is left of a long row streams through twice, the second time out of the memory-side cache.
template <int THREADS, int NV, int LV, bool GRAD>
__global__ __launch_bounds__(THREADS) void distill_row_kernel(DistillArgs g) {
    extern __shared__ __align__(16) float lds[];
    __shared__ float red[THREADS / 64][3];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const Span part(g.z + row * g.ldz, 0, g.vocab);
    f32x4* held = reinterpret_cast<f32x4*>(lds);
    constexpr int GROUP = NV < 4 ? NV : 4, FIRST = (NV + LV) * THREADS;
    // the row's entries are asked for before its logits: their own logits are then on the way behind those
    const int slots = entry_slots(g.topk);
    const Entries e = entries_at(lds + 4 * LV * THREADS, slots);
    Entry mine(g, row, tid);
    f32x4 v[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) v[i] = part.load<GRAD>(tid + i * THREADS);
    const float rest = part.rest(tid);
    if (tid < slots) mine.stage(g, e, tid, g.z + row * g.ldz, 0, g.vocab);
    for (int j = tid + THREADS; j < slots; j += THREADS) Entry(g, row, j).stage(g, e, j, g.z + row * g.ldz, 0, g.vocab);
    RowStats s = {-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; i += GROUP) {
        f32x4 u[GROUP];
#pragma unroll
        for (int q = 0; q < GROUP; q++) u[q] = v[i + q];
        stats_of(u, g.cold, g.terms, s);
        __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (LV > 0) {
#pragma unroll
        for (int i = 0; i < LV; i += 3) {
            f32x4 u[3];
#pragma unroll
            for (int q = 0; q < 3; q++) u[q] = part.load<GRAD>(tid + (NV + i + q) * THREADS);
            stats_of(u, g.cold, g.terms, s);
#pragma unroll
            for (int q = 0; q < 3; q++) held[(i + q) * THREADS + tid] = u[q];
        }
    }
    for (int at = FIRST + tid; at < part.vecs; at += 4 * THREADS) {
        f32x4 u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = part.load(at + i * THREADS);
        stats_of(u, g.cold, g.terms, s);
    }
    if (part.single(tid)) stats_of_one(rest, g.cold, s);
    s = block_stats<THREADS / 64>(s, g.cold, red);       // its barrier also publishes the entries
    float top, sum;
    teacher_softmax(g, e, top, sum);
    if (tid < 64) finish_row(g, e, s, top, sum, row);
    if (!GRAD) return;
    float* dz = g.dz + row * g.ldd + part.head;
    const GradRow r = grad_row(g, e, s, sum);
    int again = tid;                                     // the stores' offsets are computed anew, not kept since the loads
    asm volatile("" : "+v"(again));
    with_terms(g.terms, [&](auto t) {
        constexpr int TERMS = decltype(t)::value;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            grad_store<TERMS>(r, v[i], dz, again + i * THREADS, part.vecs);
            __builtin_amdgcn_sched_barrier(0);           // four gradients in registers at a time, not all
        }
        if constexpr (LV > 0) {
#pragma unroll
            for (int i = 0; i < LV; i++) {
                grad_store<TERMS>(r, held[i * THREADS + tid], dz, again + (NV + i) * THREADS, part.vecs);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        for (int at = FIRST + tid; at < part.vecs; at += 4 * THREADS) {
            f32x4 u[4];
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = part.load(at + i * THREADS);
#pragma unroll
            for (int i = 0; i < 4; i++) grad_store<TERMS>(r, u[i], dz, at + i * THREADS, part.vecs);
        }
    });
    if (part.single(tid)) dz[part.place(tid)] = grad_at(r, rest);
    __syncthreads();
    grad_entries(g, e, r, top, sum, g.dz + row * g.ldd, 0, g.vocab, THREADS);
}

// ---- rows cut into segments (37 rows of 128001 logits: 7 us for the statistics and 10 us for loss and gradient, which find the
// 38 MB in the memory-side cache; with a workgroup per row 37 of 256 compute units would work)
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
        stats_of(u, g.cold, g.terms, s);
    }
    if (part.single(threadIdx.x)) stats_of_one(part.rest(threadIdx.x), g.cold, s);
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

// the gradient of a row's segment from statistics: the segments' (with the row's loss), or those a forward call kept (8192 x 50001:
// 697 us, 4.7 TB/s, behind a forward pass of 281 us; both in one read the logits once, 673 us)
template <bool JOIN, bool GRAD>
__global__ __launch_bounds__(kSegThreads) void distill_segment_grad_kernel(DistillArgs g) {
    extern __shared__ float lds[];
    const int64_t row = blockIdx.y;
    const int begin = GRAD ? blockIdx.x * g.per_segment : 0, end = GRAD ? min(g.vocab, begin + g.per_segment) : 0;
    const float* z = g.z + row * g.ldz;
    const int slots = entry_slots(g.topk);
    const Entries e = entries_at(lds, slots);
    for (int j = threadIdx.x; j < slots; j += kSegThreads) {
        Entry x(g, row, j);
        x.stage(g, e, j, z, begin, JOIN ? 0 : end);      // only this segment's logits: others' may be overwritten already
        if (JOIN && j <= g.topk && x.index >= 0) e.logit[j] = g.seg_logit[row * (g.topk + 1) + j];
    }
    RowStats s;
    if (JOIN) s = joined_stats(g, row);
    else s = RowStats{g.stats[3 * row], g.stats[3 * row + 1], g.stats[3 * row + 2]};
    __syncthreads();
    float top, sum;
    teacher_softmax(g, e, top, sum);
    if (JOIN && blockIdx.x == 0 && threadIdx.x < 64) finish_row(g, e, s, top, sum, row);
    if (!GRAD) return;
    float* dz = g.dz + row * g.ldd;
    const GradRow r = grad_row(g, e, s, sum);
    const Span part(z, begin, end);
    with_terms(g.terms, [&](auto t) {
        for (int at = threadIdx.x; at < part.vecs; at += 4 * kSegThreads) {
            f32x4 u[4];
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = part.load(at + i * kSegThreads);
#pragma unroll
            for (int i = 0; i < 4; i++) grad_store<decltype(t)::value>(r, u[i], dz + begin + part.head, at + i * kSegThreads, part.vecs);
        }
    });
    if (part.single(threadIdx.x)) dz[begin + part.head + part.place(threadIdx.x)] = grad_at(r, part.rest(threadIdx.x));
    __syncthreads();
    grad_entries(g, e, r, top, sum, dz, begin, end, kSegThreads);
}

static int distill_check(const char* fn, const float* z, int64_t ldz, const float* teacher, const int32_t* index, int64_t rows, int64_t vocab,
                         int64_t topk, float temperature, float alpha) {
    if (rows < 0 || vocab < 1 || topk < 0) return set_error(BH_EINVAL, "%s: rows >= 0, vocab >= 1 and topk >= 0 are needed", fn);
    if (vocab > (1 << 30) || rows > (1 << 22)) return set_error(BH_EINVAL, "%s: too many rows or too large a vocabulary", fn);
    if (topk > kMaxTopk) return set_error(BH_EINVAL, "%s: topk is at most %d", fn, kMaxTopk);
    if (ldz < vocab) return set_error(BH_EINVAL, "%s: leading dimension too small", fn);
    // T^2 weighs the loss and 1/T the logits: both have to be numbers (a square of 0 would make NaN of a large divergence)
    if (!(temperature > 0.f) || !(temperature * temperature >= FLT_MIN) || !(temperature * temperature < INFINITY) ||
        !(kLog2e / temperature < INFINITY))
        return set_error(BH_EINVAL, "%s: the temperature is a positive number whose square and inverse are in range", fn);
    if (!(alpha >= 0.f && alpha <= 1.f)) return set_error(BH_EINVAL, "%s: alpha lies in [0, 1]", fn);
    if (rows > 0 && (!z || (topk > 0 && (!teacher || !index)))) return set_error(BH_EINVAL, "%s: null pointer", fn);
    return BH_OK;
}

static DistillArgs distill_args(const float* z, int64_t ldz, const float* teacher, const int32_t* index, const int32_t* labels, int64_t rows,
                                int64_t vocab, int64_t topk, float temperature, float alpha, float scale) {
    DistillArgs g = {};
    g.z = z; g.ldz = ldz; g.teacher = teacher; g.index = index; g.labels = labels;
    // a teacher without weight is not looked at: a divergence that is infinite would make 0 times infinity of it
    g.rows = rows; g.vocab = (int)vocab; g.topk = alpha == 0.f ? 0 : (int)topk;
    g.inv_t = 1.f / temperature;
    g.cold = kLog2e / temperature;
    g.w_soft = alpha * temperature * temperature;
    g.w_hard = labels ? 1.f - alpha : 0.f;
    g.terms = g.w_hard == 0.f ? kSoft : temperature == 1.f ? kSame : kBoth;
    g.g_soft = scale * alpha * temperature;
    g.g_hard = scale * (1.f - alpha);
    return g;
}

// segments of a row so that a few rows still fill the chip; 1 = a workgroup per row.  Loss and gradient, us, in segments / a
// workgroup per row: 16 rows of 32000 12 / 18, 64 of 50001 15 / 17, 64 of 128001 24 / 31, 128 of 32000 17 / 18; 64 of 12000 15 / 13,
// 16 of 8192 14 / 9, 128 of 50001 21 / 19, 200 of 50001 32 / 25, 255 of 128001 69 / 64.
static int segments_for(int64_t rows, int64_t vocab) {
    if (rows >= 128 || vocab < 16384) return 1;
    const int64_t want = ceil_div(512, rows), most = ceil_div(vocab, 4096);
    return (int)(want < most ? want : most);
}
static void cut_row(DistillArgs& g, int segments) {
    g.per_segment = (int)(ceil_div(ceil_div(g.vocab, segments), 4) * 4);
    g.segments = (int)ceil_div(g.vocab, g.per_segment);
}

template <int THREADS, int NV, int LV, bool GRAD>
static int launch_row_kernel(const DistillArgs& g) {
    const auto bytes = [](int topk) { return sizeof(float) * (4 * (size_t)LV * THREADS + 3 * (size_t)entry_slots(topk)); };
    static bool raised = false;                  // the most that any call needs, so that two threads may both ask for it
    if (!raised && bytes(kMaxTopk) > 64 * 1024) {
        const int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(&distill_row_kernel<THREADS, NV, LV, GRAD>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes(kMaxTopk)), "bh_distill: LDS size");
        if (rc) return rc;
        raised = true;
    }
    hipLaunchKernelGGL((distill_row_kernel<THREADS, NV, LV, GRAD>), dim3((unsigned)g.rows), dim3(THREADS), bytes(g.topk), stream(), g);
    return BH_LAUNCH_CHECK("bh_distill");
}

// Threads and registers per row, by the row's length: a row that fits wholly is read once; with 512 threads and LDS two rows of
// 51 K logits share a compute unit, one being read while the other is worked on.  Loss and gradient on 4096 to 16384 rows, us:
//   758 logits   17 with 64 x 4 vectors, 20 with 128 x 4, 26 with 256 x 4      2000   54 with 128 x 4, 59 with 256 x 4
//   8000   213 with 256 x 8, 236 with 512 x 8      16000   200 with 512 x 8, 221 with 256 x 8, 246 with LDS
//   32000  194 with LDS, 205 with 512 x 8          50001   683 with LDS, 761 with 512 x 8, 810 with 1024 x 8
// The loss alone reads the row once anyway.
template <bool GRAD>
static int launch_rows(const DistillArgs& g) {
    if (g.vocab <= 1024) return launch_row_kernel<64, 4, 0, GRAD>(g);
    if (g.vocab <= 2048) return launch_row_kernel<128, 4, 0, GRAD>(g);
    if (g.vocab <= 4096) return launch_row_kernel<256, 4, 0, GRAD>(g);
    if (!GRAD) return launch_row_kernel<512, 8, 0, GRAD>(g);
    if (g.vocab <= 8192) return launch_row_kernel<256, 8, 0, true>(g);
    if (g.vocab <= 24576) return launch_row_kernel<512, 8, 0, true>(g);
    return launch_row_kernel<512, 16, 9, true>(g);
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
        const size_t lds = sizeof(float) * 3 * (size_t)entry_slots(g.topk);
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
    // a workgroup streams a segment of at most 16 K logits, of at least 4 K where rows are few (nothing has to be joined here); the
    // grid's second dimension holds 65535 rows
    const int64_t by_size = ceil_div(vocab, 16384), most = ceil_div(vocab, 4096), want = ceil_div(512, rows), by_rows = want < most ? want : most;
    cut_row(g, (int)(by_size > by_rows ? by_size : by_rows));
    const size_t lds = sizeof(float) * 3 * (size_t)entry_slots((int)topk);
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
