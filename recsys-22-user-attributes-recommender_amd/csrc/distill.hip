// Distillation from a teacher's best items: the KL divergence of the student's full-catalogue softmax from the teacher's
// distribution over its own short list, and its gradient, next to CrossEntropyLoss over the same logits (heads.hip).
//
//   list of row r: the entries j with 0 <= ids[r][j] < V;  p = softmax over the list of t[r][j] / tau
//   q = softmax over the catalogue of s[r][v] / tau
//   loss = w * mean over the rows with a list of  tau^2 sum_j p_j (log p_j - log q_{id_j})
//   dL/ds[r][v] = w tau / rows with a list * (q_v - sum_{j: id_j = v} p_j)
//
// Two schedules, both memory bound.
//   apart: one pass over the logits forward (running maximum and sum in base-2 exponentials), one read and one write
//   backward: 3 n V elements, for any row.
//   together (asme_distill_xent_fwd_grad): a workgroup holds its row in registers, so that the forward writes the gradient
//   of the mean as well: the 2 n V elements that any schedule has to move.  The backward has the upstream factor left to
//   apply, which costs nothing where it is 1 and 2 n V more where it is not: a loss that is one part of another takes its
//   weight w here.  fp32 is then scaled in place (a second rounding of 2^-24, below what the row's sum leaves); bf16 is
//   formed anew from the logits, since scaling would round it to 8 bits twice.
// Rows are split over workgroups when there are fewer rows than the chip needs workgroups; the splits' (maximum, sum) pairs
// are merged in a fixed order, so a schedule's results repeat bit for bit (the two differ in the order of their sums).
// Statistics, probabilities and the loss are fp32; a bf16 gradient is rounded once, on store.
// Measured: together, 8192 x 26747 fp32 with lists of 50, 372 us forward and backward -- 1758 MB at 4.7 TB/s, what a copy
// reaches on this card; apart, 580 us.  64 x 10007 bf16: 30 us of kernels, of 110 that the calls and autograd take.
#include "elem.h"

using namespace asme;

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;           // 16-byte vectors in flight per thread
constexpr int kMaxTop = 1024;        // entries of a teacher list
constexpr int kMaxSplits = 64;       // one lane of the merging wave each
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// workgroups per row: enough for eight per CU, each at least 4096 elements (16 per thread)
int row_splits(int64_t n, int64_t V) {
    const int64_t want = (2048 + n - 1) / n, most = (V + 4095) / 4096;
    return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxSplits}));
}
// elements per split: a multiple of 64, so the splits differ by at most that
int64_t split_len(int64_t V, int splits) { return ((V + splits - 1) / splits + 63) / 64 * 64; }

struct MaxSum {
    float m, s;  // s = sum of 2^(x - m)
};
__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b) {
    const float m = fmaxf(a.m, b.m), base = m == -INFINITY ? 0.f : m;
    return {m, a.s * exp2f(a.m - base) + b.s * exp2f(b.m - base)};
}
__device__ __forceinline__ MaxSum wave_merge(MaxSum a) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) a = merge(a, {__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64)});
    return a;
}

// NE more elements into a running (maximum, sum)
template <int NE>
__device__ __forceinline__ void take(MaxSum& a, const float (&x)[NE], float scale) {
    float t = x[0];
#pragma unroll
    for (int i = 1; i < NE; ++i) t = fmaxf(t, x[i]);
    t *= scale;
    if (t > a.m) {
        a.s *= __builtin_amdgcn_exp2f(a.m - t);
        a.m = t;
    }
    const float base = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int i = 0; i < NE; ++i) a.s += __builtin_amdgcn_exp2f(fmaf(x[i], scale, -base));
}

// a row segment [p, p + len) as an unaligned head, whole 16-byte vectors and a tail
template <class T>
struct Segment {
    int64_t head, vecs;
    __device__ Segment(const T* p, int64_t len) {
        const int64_t off = (int64_t)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T));
        head = off < len ? off : len;
        vecs = (len - head) / Elem<T>::V;
    }
};

template <class T>
__global__ __launch_bounds__(kThreads) void stats_kernel(const T* __restrict__ logits, int64_t ld, int64_t V,
                                                         int splits, int64_t seg_len, float scale,
                                                         MaxSum* __restrict__ part) {
    constexpr int E = Elem<T>::V;
    const int64_t row = blockIdx.x / splits;
    const int64_t begin = (int64_t)(blockIdx.x % splits) * seg_len;
    const int64_t len = max((int64_t)0, min(seg_len, V - begin));
    const T* p = logits + row * ld + begin;
    const Segment<T> sg(p, len);
    MaxSum a{-INFINITY, 0.f};
    const T* body = p + sg.head;
    int64_t i = threadIdx.x;
    for (; i + (kUnroll - 1) * kThreads < sg.vecs; i += kUnroll * kThreads) {
        float x[kUnroll][E];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) Elem<T>::load(body + (i + u * kThreads) * E, x[u]);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) take(a, x[u], scale);
    }
    for (; i < sg.vecs; i += kThreads) {
        float x[E];
        Elem<T>::load(body + i * E, x);
        take(a, x, scale);
    }
    const int64_t tail = sg.head + sg.vecs * E;  // head and tail: fewer than 16 elements together
    for (int64_t j = threadIdx.x; j < sg.head + len - tail; j += kThreads) {
        const float x[1] = {Elem<T>::get(p + (j < sg.head ? j : tail + j - sg.head))};
        take(a, x, scale);
    }
    a = wave_merge(a);
    __shared__ MaxSum w[kThreads / 64];
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kThreads / 64; ++k) a = merge(a, w[k]);
        part[blockIdx.x] = a;
    }
}

// The wave's maximum of a list's present logits; `there`: the row has a list -- a present entry above -infinity, or a NaN,
// which the maximum skips and which is to reach the loss
__device__ __forceinline__ float list_max(const int64_t* id, const float* t, int top, int64_t V, bool& there) {
    float m = -INFINITY;
    bool any = false;
    for (int j = threadIdx.x & 63; j < top; j += 64)
        if ((uint64_t)id[j] < (uint64_t)V) {
            m = fmaxf(m, t[j]);
            any = any || !(t[j] == -INFINITY);
        }
    there = __any(any);
    return wave_max(m);
}

// One wave per row: its softmax state (maximum in base 2, 1 / sum; 0 for a row without a list) -- kept apart, since
// lse rounded to fp32 would cost every q of the row |lse| 2^-24 --, p (n x top, 0 for absent entries), and the workgroup's (loss,
// rows) sums in the order of its waves; `finish` (one workgroup in all): the mean at once.
template <class T>
__global__ __launch_bounds__(1024) void rows_kernel(const T* __restrict__ logits, int64_t ld, int64_t n, int64_t V,
                                                    const int64_t* __restrict__ ids, const float* __restrict__ teacher,
                                                    int top, float scale, float inv_tau, float tau2, int splits,
                                                    const MaxSum* __restrict__ part, float2* __restrict__ state,
                                                    float* __restrict__ prob, float* __restrict__ sums, int finish,
                                                    float* __restrict__ out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    float loss = 0.f, rows = 0.f;
    for (int64_t row = (int64_t)blockIdx.x * waves + wave; row < n; row += (int64_t)gridDim.x * waves) {
        MaxSum a{-INFINITY, 0.f};
        if (lane < splits) a = part[row * splits + lane];
        a = wave_merge(a);
        const float log_s = logf(a.s);
        const int64_t* id = ids + row * top;
        const float* t = teacher + row * top;
        bool there;
        const float tm = list_max(id, t, top, V, there);
        float ts = 0.f;
        for (int j = lane; j < top; j += 64)
            if ((uint64_t)id[j] < (uint64_t)V && there) ts += expf((t[j] - tm) * inv_tau);
        ts = wave_sum(ts);
        const float log_ts = logf(ts);
        float kl = 0.f;
        for (int j = lane; j < top; j += 64) {
            const int64_t v = id[j];
            float pj = 0.f;
            if (there && (uint64_t)v < (uint64_t)V) {
                const float lp = (t[j] - tm) * inv_tau - log_ts;
                pj = expf((t[j] - tm) * inv_tau) / ts;  // (not of lp, whose rounding grows with the list's length)
                if (!(pj == 0.f)) kl += pj * (lp - (fmaf(Elem<T>::get(logits + row * ld + v), scale, -a.m) * kLn2 - log_s));
            }
            prob[row * top + j] = pj;
        }
        kl = wave_sum(kl);
        if (lane == 0) state[row] = make_float2(there ? a.m : 0.f, there ? 1.f / a.s : 0.f);
        loss += there ? kl * tau2 : 0.f;
        rows += there ? 1.f : 0.f;
    }
    __shared__ float w[2][16];
    if (lane == 0) {
        w[0][wave] = loss;
        w[1][wave] = rows;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < waves; ++k) {
            loss += w[0][k];
            rows += w[1][k];
        }
        if (finish) {
            out[0] = loss / rows;  // no row with a list: NaN, as the mean over no rows
            out[1] = rows;
        } else {
            sums[2 * blockIdx.x] = loss;
            sums[2 * blockIdx.x + 1] = rows;
        }
    }
}

__global__ __launch_bounds__(1024) void mean_kernel(const float* __restrict__ sums, int64_t n, float* __restrict__ out) {
    float loss = 0.f, rows = 0.f;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        loss += sums[2 * i];
        rows += sums[2 * i + 1];
    }
    loss = wave_sum(loss);
    rows = wave_sum(rows);
    __shared__ float w[2][16];
    if ((threadIdx.x & 63) == 0) {
        w[0][threadIdx.x >> 6] = loss;
        w[1][threadIdx.x >> 6] = rows;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 16; ++k) {
            loss += w[0][k];
            rows += w[1][k];
        }
        out[0] = loss / rows;
        out[1] = rows;
    }
}

// One wave per row: p (n x top), and the workgroup's number of rows with a list
__global__ __launch_bounds__(1024) void teacher_kernel(const int64_t* __restrict__ ids, const float* __restrict__ teacher,
                                                       int64_t n, int64_t V, int top, float inv_tau,
                                                       float* __restrict__ prob, float* __restrict__ counts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * 16 + wave;
    bool there = false;
    if (row < n) {
        const int64_t* id = ids + row * top;
        const float* t = teacher + row * top;
        float ts = 0.f;
        const float tm = list_max(id, t, top, V, there);
        for (int j = lane; j < top; j += 64)
            if (there && (uint64_t)id[j] < (uint64_t)V) ts += expf((t[j] - tm) * inv_tau);
        ts = wave_sum(ts);
        for (int j = lane; j < top; j += 64)
            prob[row * top + j] = there && (uint64_t)id[j] < (uint64_t)V ? expf((t[j] - tm) * inv_tau) / ts : 0.f;
    }
    __shared__ float w[16];
    if (lane == 0) w[wave] = there ? 1.f : 0.f;
    __syncthreads();
    if (threadIdx.x == 0) {
        float c = 0.f;
        for (int k = 0; k < 16; ++k) c += w[k];
        counts[2 * blockIdx.x] = 0.f;
        counts[2 * blockIdx.x + 1] = c;
    }
}

constexpr int kRowThreads = 512, kMostVecs = 16;  // 16-byte vectors a thread: rows to 32 K fp32 or 64 K bf16 items

// A whole row per workgroup: its state, its loss and the gradient of the mean (stats[1]: the rows with a list).  Two
// or three workgroups a CU, so that one's loads are on their way while another reduces.
template <class T, int kRowVecs>
__global__ __launch_bounds__(kRowThreads, kRowVecs == kMostVecs ? 4 : 6) void fused_kernel(const T* __restrict__ logits, int64_t ld, int V,
                                                               const int64_t* __restrict__ ids, int top, float scale,
                                                               float tau2, float tau1, const float* __restrict__ prob,
                                                               const float* __restrict__ stats,
                                                               float2* __restrict__ state, float* __restrict__ sums,
                                                               T* __restrict__ dlogits, int64_t ld_d) {
    constexpr int E = Elem<T>::V;
    typedef T Vec __attribute__((ext_vector_type(E)));
    __shared__ int list[kMaxTop];
    __shared__ float lp[kMaxTop];
    __shared__ float red[2][kRowThreads / 64];
    const int64_t row = blockIdx.x;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const T* p = logits + row * ld;
    T* d = dlogits + row * ld_d;
    // whole vectors, and the elements before and behind them: fewer than 16, one a thread
    const int head = (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T)), vecs = (V - head) / E, tail = head + vecs * E;
    const int edge = t < head ? t : tail + t - head;
    const bool has_edge = t < head + V - tail;
    // (a thread's vectors: t, t + 512, ...; behind the row its last one again)
    Vec raw[kRowVecs];
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u)
        raw[u] = reinterpret_cast<const Vec*>(p + head)[(unsigned)min(t + u * kRowThreads, vecs - 1)];
    const float ex = has_edge ? Elem<T>::get(p + edge) : -INFINITY;
    float listed = 0.f;
    for (int j = t; j < top; j += kRowThreads) {
        const int64_t v = ids[row * top + j];
        list[j] = (uint64_t)v < (uint64_t)V ? (int)v : -1;
        lp[j] = prob[row * top + j];
        listed += lp[j];
    }
    // the row stays as it is stored: without this the compiler keeps a bf16 row's values as floats from one pass over it to
    // the next, twice the registers
    auto stored = [&]() {
#pragma unroll
        for (int u = 0; u < kRowVecs; ++u) {
            floatx4 v = __builtin_bit_cast(floatx4, raw[u]);
            asm volatile("" : "+v"(v));
            raw[u] = __builtin_bit_cast(Vec, v);
        }
    };
    float m = ex;  // (a vector seen twice does not change the maximum)
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, (float)raw[u][e]);
    m = wave_max(m);
    listed = wave_sum(listed);
    if (lane == 0) red[0][wave] = m, red[1][wave] = listed;
    __syncthreads();
    m = red[0][0], listed = red[1][0];
    for (int k = 1; k < kRowThreads / 64; ++k) m = fmaxf(m, red[0][k]), listed += red[1][k];
    m *= scale;
    const bool there = listed != 0.f;  // a list's p sum to 1; no list, no p (a NaN goes on)
    const float base = m == -INFINITY ? 0.f : m;
    float s = __builtin_amdgcn_exp2f(fmaf(ex, scale, -base));
    stored();
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u) {
        float part = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) part += __builtin_amdgcn_exp2f(fmaf((float)raw[u][e], scale, -base));
        s += t + u * kRowThreads < vecs ? part : 0.f;
    }
    s = wave_sum(s);
    __syncthreads();
    if (lane == 0) red[0][wave] = s;
    __syncthreads();
    s = red[0][0];
    for (int k = 1; k < kRowThreads / 64; ++k) s += red[0][k];
    const float inv = there ? 1.f / s : 0.f, g = there ? tau1 / stats[1] : 0.f, log_s = logf(s);
    auto q = [&](float x) { return there ? __builtin_amdgcn_exp2f(fmaf(x, scale, -base)) * inv : 0.f; };
    stored();
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u)
        if (t + u * kRowThreads < vecs) {
            Vec o;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = (T)(g * q((float)raw[u][e]));
            reinterpret_cast<Vec*>(d + head)[(unsigned)(t + u * kRowThreads)] = o;
        }
    if (has_edge) Elem<T>::put(d + edge, g * q(ex));
    __syncthreads();  // the list's entries are stored after the row
    float kl = 0.f;
    for (int j = t; j < top; j += kRowThreads) {
        const int v = list[j];
        if (v < 0 || !there) continue;
        const float x = Elem<T>::get(p + v);
        if (!(lp[j] == 0.f)) kl += lp[j] * (logf(lp[j]) - (fmaf(x, scale, -base) * kLn2 - log_s));
        float sum = 0.f;
        bool first = true;
        for (int k = 0; k < top; ++k) {
            const bool same = list[k] == v;
            first = first && !(same && k < j);
            sum += same ? lp[k] : 0.f;
        }
        if (first) Elem<T>::put(d + v, g * (q(x) - sum));
    }
    kl = wave_sum(kl);
    if (lane == 0) red[1][wave] = kl;  // (last read before the barrier above)
    __syncthreads();
    if (t == 0) {
        for (int k = 1; k < kRowThreads / 64; ++k) kl += red[1][k];
        state[row] = make_float2(there ? base : 0.f, inv);
        sums[2 * row] = there ? kl * tau2 : 0.f;
        sums[2 * row + 1] = there ? 1.f : 0.f;
    }
}

// x *= f[0], nothing where that is 1
template <class T>
__global__ __launch_bounds__(kThreads) void scale_kernel(T* __restrict__ x, int64_t n, const float* __restrict__ f) {
    constexpr int E = Elem<T>::V;
    const float g = f[0];
    if (g == 1.f) return;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n / E; i += (int64_t)gridDim.x * kThreads) {
        float v[E];
        Elem<T>::load(x + i * E, v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] *= g;
        Elem<T>::store(x + i * E, v);
    }
    const int64_t j = n / E * E + threadIdx.x;
    if (blockIdx.x == 0 && j < n) Elem<T>::put(x + j, Elem<T>::get(x + j) * g);
}

// dlogits of a row segment: g (q - 0) everywhere, then the list's entries of the segment once more with their p taken
// off.  An item that is on the list twice is written by its first entry, with the sum of its p in list order.  `again`:
// dlogits holds the gradient for dloss = 1 already, and nothing is left to do where it is 1.
template <class T>
__global__ __launch_bounds__(kThreads) void grad_kernel(const T* __restrict__ logits, int64_t ld, int64_t V,
                                                        const int64_t* __restrict__ ids, int top, int splits,
                                                        int64_t seg_len, float scale, float tau,
                                                        const float2* __restrict__ state,
                                                        const float* __restrict__ prob,
                                                        const float* __restrict__ stats,
                                                        const float* __restrict__ dloss, int again,
                                                        T* __restrict__ dlogits, int64_t ld_d) {
    constexpr int E = Elem<T>::V;
    __shared__ int list[kMaxTop];
    __shared__ float lp[kMaxTop];
    if (again && dloss[0] == 1.f) return;  // (the whole grid)
    const int64_t row = blockIdx.x / splits;
    const int64_t begin = (int64_t)(blockIdx.x % splits) * seg_len;
    const int64_t len = max((int64_t)0, min(seg_len, V - begin));
    const T* p = logits + row * ld + begin;
    T* d = dlogits + row * ld_d + begin;
    const float2 st = state[row];
    const bool there = !(st.y == 0.f);
    const float g = there ? dloss[0] * tau / stats[1] : 0.f;
    for (int j = threadIdx.x; j < top; j += kThreads) {
        const int64_t v = ids[row * top + j] - begin;
        list[j] = there && v >= 0 && v < len ? (int)v : -1;
        lp[j] = prob[row * top + j];
    }
    auto q = [&](float x) { return there ? __builtin_amdgcn_exp2f(fmaf(x, scale, -st.x)) * st.y : 0.f; };
    const Segment<T> sg(p, len);
    const int64_t tail = sg.head + sg.vecs * E;
    if (((uintptr_t)(d + sg.head) & 15) == 0) {
        const T* body = p + sg.head;
        int64_t i = threadIdx.x;
        for (; i + (kUnroll - 1) * kThreads < sg.vecs; i += kUnroll * kThreads) {
            float x[kUnroll][E];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) Elem<T>::load(body + (i + u * kThreads) * E, x[u]);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
                for (int e = 0; e < E; ++e) x[u][e] = g * q(x[u][e]);
                Elem<T>::store(d + sg.head + (i + u * kThreads) * E, x[u]);
            }
        }
        for (; i < sg.vecs; i += kThreads) {
            float x[E];
            Elem<T>::load(body + i * E, x);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = g * q(x[e]);
            Elem<T>::store(d + sg.head + i * E, x);
        }
        for (int64_t j = threadIdx.x; j < sg.head + len - tail; j += kThreads) {
            const int64_t v = j < sg.head ? j : tail + j - sg.head;
            Elem<T>::put(d + v, g * q(Elem<T>::get(p + v)));
        }
    } else {  // the two rows are aligned differently: element by element
        for (int64_t v = threadIdx.x; v < len; v += kThreads) Elem<T>::put(d + v, g * q(Elem<T>::get(p + v)));
    }
    __syncthreads();  // the list is in LDS, and its entries are stored after the whole segment
    for (int j = threadIdx.x; j < top; j += kThreads) {
        const int v = list[j];
        if (v < 0) continue;
        float sum = 0.f;
        bool first = true;
        for (int k = 0; k < top; ++k) {
            const bool same = list[k] == v;
            first = first && !(same && k < j);
            sum += same ? lp[k] : 0.f;
        }
        if (first) Elem<T>::put(d + v, g * (q(Elem<T>::get(p + v)) - sum));
    }
}

constexpr int64_t kOneGroupRows = 256;  // up to here one workgroup finishes the rows and their mean
int64_t finish_groups(int64_t n) { return n <= kOneGroupRows ? 1 : (n + 15) / 16; }

// the rows that a workgroup holds, where there are enough of them to fill the chip (two workgroups a CU; 424 us for
// 8192 x 26747 fp32 at 1024 threads of 64 registers, which spilled, 355 at 512 of 128)
bool together(int64_t n, int64_t V, int dtype) {
    return n >= 512 && V >= 4096 && V <= (int64_t)kRowThreads * kMostVecs * (dtype == kF32 ? 4 : 8);
}

bool shape_ok(int64_t n, int64_t V, int64_t top) {
    return n >= 0 && n < (1ll << 24) && V >= 1 && V < (1ll << 31) && top >= 1 && top <= kMaxTop;
}

}  // namespace

ASME_API int64_t asme_distill_xent_workspace(int64_t n, int64_t V) {
    if (n < 1 || !shape_ok(n, V, 1)) return 0;
    return n * row_splits(n, V) * (int64_t)sizeof(MaxSum) + finish_groups(n) * 8;
}

ASME_API int asme_distill_xent_fwd(const void* logits, int64_t ld, int64_t n, int64_t V, const int64_t* ids,
                                   const float* teacher, int64_t top, float temperature, float weight, int dtype,
                                   float* state, float* prob, void* workspace, int64_t ws_bytes, float* out, void* stream) {
    ASME_CHECK_ARG(logits && ids && teacher && state && prob && workspace && out, "asme_distill_xent_fwd: null pointer");
    ASME_CHECK_ARG(dtype_ok(dtype), "asme_distill_xent_fwd: dtype is 0 (fp32) or 1 (bf16)");
    ASME_CHECK_ARG(n >= 1 && shape_ok(n, V, top) && ld >= V, "asme_distill_xent_fwd: bad size");
    ASME_CHECK_ARG(temperature > 0.f && temperature < INFINITY && weight - weight == 0.f,
                   "asme_distill_xent_fwd: temperature > 0, a finite weight");
    ASME_CHECK_ARG(ws_bytes >= asme_distill_xent_workspace(n, V), "asme_distill_xent_fwd: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    const int splits = row_splits(n, V);
    const int64_t groups = finish_groups(n);
    MaxSum* part = (MaxSum*)workspace;
    float* sums = (float*)(part + n * splits);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL(stats_kernel<T>, dim3((unsigned)(n * splits)), dim3(kThreads), 0, s, (const T*)logits, ld, V,
                           splits, split_len(V, splits), kLog2e / temperature, part);
        hipLaunchKernelGGL(rows_kernel<T>, dim3((unsigned)groups), dim3(1024), 0, s, (const T*)logits, ld, n, V, ids,
                           teacher, (int)top, kLog2e / temperature, 1.f / temperature, weight * temperature * temperature, splits,
                           part, (float2*)state, prob,
                           sums, groups == 1, out);
    });
    if (groups > 1) hipLaunchKernelGGL(mean_kernel, dim3(1), dim3(1024), 0, s, sums, groups, out);
    ASME_LAUNCH_CHECK("asme_distill_xent_fwd");
}

ASME_API int asme_distill_xent_grad_supported(int64_t n, int64_t V, int dtype) {
    return dtype_ok(dtype) && n >= 1 && shape_ok(n, V, 1) && together(n, V, dtype);
}
ASME_API int64_t asme_distill_xent_grad_workspace(int64_t n) { return n >= 1 && shape_ok(n, 1, 1) ? n * 8 + (n + 15) / 16 * 8 : 0; }

// The forward with the gradient of the mean (before the upstream factor): dlogits contiguous, its rows aligned like those
// of logits.
ASME_API int asme_distill_xent_fwd_grad(const void* logits, int64_t ld, int64_t n, int64_t V, const int64_t* ids,
                                        const float* teacher, int64_t top, float temperature, float weight, int dtype,
                                        float* state, float* prob, void* dlogits, void* workspace, int64_t ws_bytes, float* out,
                                        void* stream) {
    ASME_CHECK_ARG(logits && ids && teacher && state && prob && dlogits && workspace && out,
                   "asme_distill_xent_fwd_grad: null pointer");
    ASME_CHECK_ARG(logits != dlogits, "asme_distill_xent_fwd_grad: dlogits must not be logits");
    ASME_CHECK_ARG(n >= 1 && shape_ok(n, V, top) && ld >= V && asme_distill_xent_grad_supported(n, V, dtype),
                   "asme_distill_xent_fwd_grad: bad size");
    ASME_CHECK_ARG(((uintptr_t)logits & 15) == ((uintptr_t)dlogits & 15) && (ld - V) * dtype_size(dtype) % 16 == 0,
                   "asme_distill_xent_fwd_grad: rows of logits and dlogits are aligned alike");
    ASME_CHECK_ARG(temperature > 0.f && temperature < INFINITY && weight - weight == 0.f,
                   "asme_distill_xent_fwd_grad: temperature > 0, a finite weight");
    ASME_CHECK_ARG(ws_bytes >= asme_distill_xent_grad_workspace(n), "asme_distill_xent_fwd_grad: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    float* sums = (float*)workspace;
    float* counts = sums + 2 * n;
    const int64_t groups = (n + 15) / 16;
    hipLaunchKernelGGL(teacher_kernel, dim3((unsigned)groups), dim3(1024), 0, s, ids, teacher, n, V, (int)top,
                       1.f / temperature, prob, counts);
    hipLaunchKernelGGL(mean_kernel, dim3(1), dim3(1024), 0, s, counts, groups, out);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        auto launch = [&](auto vecs) {
            hipLaunchKernelGGL((fused_kernel<T, decltype(vecs)::value>), dim3((unsigned)n), dim3(kRowThreads), 0, s,
                               (const T*)logits, ld, (int)V, ids, (int)top, kLog2e / temperature,
                               weight * temperature * temperature, weight * temperature, prob, out, (float2*)state, sums,
                               (T*)dlogits, V);
        };
        if (V <= kRowThreads * kMostVecs / 2 * Elem<T>::V) launch(std::integral_constant<int, kMostVecs / 2>{});
        else launch(std::integral_constant<int, kMostVecs>{});
    });
    hipLaunchKernelGGL(mean_kernel, dim3(1), dim3(1024), 0, s, sums, n, out);
    ASME_LAUNCH_CHECK("asme_distill_xent_fwd_grad");
}

// x (n values, 16-byte aligned) *= factor[0]
ASME_API int asme_scale_by(void* x, int64_t n, int dtype, const float* factor, void* stream) {
    ASME_CHECK_ARG(x && factor, "asme_scale_by: null pointer");
    ASME_CHECK_ARG(dtype_ok(dtype) && n >= 0 && ((uintptr_t)x & 15) == 0, "asme_scale_by: bad argument");
    if (n == 0) return 0;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t groups = (n / Elem<T>::V + kThreads - 1) / kThreads;
        hipLaunchKernelGGL(scale_kernel<T>, dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(groups, 4096))),
                           dim3(kThreads), 0, (hipStream_t)stream, (T*)x, n, factor);
    });
    ASME_LAUNCH_CHECK("asme_scale_by");
}

static int distill_bwd(const void* logits, int64_t ld, int64_t n, int64_t V, const int64_t* ids, int64_t top,
                       float temperature, float weight, int dtype, const float* state, const float* prob,
                       const float* stats, const float* dloss, int again, void* dlogits, int64_t ld_d, void* stream) {
    ASME_CHECK_ARG(logits && ids && state && prob && stats && dloss && dlogits, "asme_distill_xent_bwd: null pointer");
    ASME_CHECK_ARG(logits != dlogits, "asme_distill_xent_bwd: dlogits must not be logits");
    ASME_CHECK_ARG(dtype_ok(dtype), "asme_distill_xent_bwd: dtype is 0 (fp32) or 1 (bf16)");
    ASME_CHECK_ARG(n >= 1 && shape_ok(n, V, top) && ld >= V && ld_d >= V, "asme_distill_xent_bwd: bad size");
    ASME_CHECK_ARG(temperature > 0.f && temperature < INFINITY && weight - weight == 0.f,
                   "asme_distill_xent_bwd: temperature > 0, a finite weight");
    const int splits = row_splits(n, V);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL(grad_kernel<T>, dim3((unsigned)(n * splits)), dim3(kThreads), 0, (hipStream_t)stream,
                           (const T*)logits, ld, V, ids, (int)top, splits, split_len(V, splits), kLog2e / temperature,
                           weight * temperature, (const float2*)state, prob, stats, dloss, again, (T*)dlogits, ld_d);
    });
    ASME_LAUNCH_CHECK("asme_distill_xent_bwd");
}

ASME_API int asme_distill_xent_bwd(const void* logits, int64_t ld, int64_t n, int64_t V, const int64_t* ids, int64_t top,
                                   float temperature, float weight, int dtype, const float* state, const float* prob,
                                   const float* stats, const float* dloss, void* dlogits, int64_t ld_d, void* stream) {
    return distill_bwd(logits, ld, n, V, ids, top, temperature, weight, dtype, state, prob, stats, dloss, 0, dlogits, ld_d,
                       stream);
}

// What is left to do behind asme_distill_xent_fwd_grad: dlogits (contiguous) formed anew where dloss is not 1
ASME_API int asme_distill_xent_bwd_again(const void* logits, int64_t ld, int64_t n, int64_t V, const int64_t* ids,
                                         int64_t top, float temperature, float weight, int dtype, const float* state,
                                         const float* prob, const float* stats, const float* dloss, void* dlogits,
                                         void* stream) {
    return distill_bwd(logits, ld, n, V, ids, top, temperature, weight, dtype, state, prob, stats, dloss, 1, dlogits, V,
                       stream);
}
