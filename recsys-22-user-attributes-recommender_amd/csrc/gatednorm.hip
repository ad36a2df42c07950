// The end of one block and the start of the next in one pass, next to residual + LayerNorm (norm.hip): the block's output
// normed, gated and added to a scaled residual, and the sum normed for the next block.
//
//   branch = Npost(y);  s = a * res + gate * branch;  z = Npre(s)
//   N(x) = (x - mean) r * w + b, r = 1 / sqrt(var + eps);  root-mean-square form: mean = 0, r = 1 / sqrt(mean x^2 + eps)
//   backward of (ds, dz), x^ the normalised rows of y (post) and s (pre):
//     d    = ds + Npre'(dz);          Npre'(g) = r (h - mean(h) - x^ mean(h x^)), h = g w (rms: without mean(h))
//     dres = a d;  dgate = d * branch;  dy = Npost'(d * gate);  dw, db: column sums of g x^ and g
//
// gate: none, or one row of `dim` values for every rows_per_gate consecutive rows (all rows: a gate per channel; one
// sequence's rows: a gate per sequence; 1: a gate per element).
// Memory bound: forward reads res, y and writes s, z; backward reads res, y, ds, dz and writes dres, dy (s is formed
// again from res and y, in fp32, instead of being read back rounded).  A row is held in registers, one 16-byte vector a
// thread (16 .. 1024 threads: a row's sums are lane moves within a wave, and one LDS exchange beyond it), and the next row
// is on its way during its sums.  Weights stay in registers over a workgroup's rows.  Column sums: registers
// (LDS beyond 4096 columns) over a workgroup's rows, then partial rows summed in a fixed order -- no atomics.
// Measured (forward, whose four tensors are read or written once, and backward, whose six are): 16384 x 4096 bf16, a gate
// per channel, 124 us for 537 MB (4.3 TB/s) and 220 for 805 (3.7); 204800 x 128 fp32, a gate per sequence or channel, 81 us
// for 419 MB (5.2; a part comes from the cache) and 144 for 629 (4.4).  Rows that are not whole vectors, with a gate per
// channel, take 1.6 to 3 times the copy rate's time: 3479 x 6299 bf16 101 + 121 us for 175 + 263 MB, 4050 x 2922 bf16 55 + 78
// for 95 + 142, 303858 x 67 fp32 127 + 202 for 326 + 489; so do rows just beyond 4096 columns, 6710 x 4144 fp32 141 + 217 for
// 445 + 667, where half of the 1024 threads hold nothing of the second vector.
#include "elem.h"

using namespace asme;

namespace {

constexpr int kMaxDim = 8192;

// A row over TPR threads of N values each, in vectors of 16 bytes.  EVEN: rows are whole vectors on their boundaries; else
// vectors begin anywhere (global memory is read and written at any address) and the last one, part of a vector, goes
// element by element -- a branch around a row's loads that costs even rows 8 % (16384 x 4096 bf16, backward: 211 us
// without, 228 with it), but rows of 1024 threads less than the registers it saves (8192 x 4096 fp32: 333 us with it, 435
// without), which therefore always take it.
template <class T, int TPR, int N, bool EVEN>
struct Row {
    static constexpr int kPer = N, TPRv = TPR;
    static constexpr int kThreads = TPR > 64 ? TPR : 256;
    static constexpr int kSlots = kThreads / TPR;  // rows at a time
    static constexpr int E = Elem<T>::V, kVecs = N / E;
    // rows beyond 4096 values: the backward's column sums of the weights' gradients are held in LDS (128 KiB, a thread's own
    // vectors) and its rows read when they are due; beside them in 128 registers they spilled up to 173 values (forward and
    // backward, 4000 x 8192 fp32: 473 us, 303 with the sums in LDS; 2 x 2000 x 8192 bf16, a gate a row: 546, 254)
    static constexpr bool kLean = TPR * N > 4096;
    typedef T Vec __attribute__((ext_vector_type(E)));
    typedef Vec AnyVec __attribute__((aligned(EVEN ? 16 : sizeof(T))));
    // a row's values as they are stored
    struct Raw {
        Vec v[kVecs];
        template <bool WHOLE>
        __device__ __forceinline__ void load(const T* p, int t, int D, int c) {  // its vector c
            const int j = (c * TPR + t) * E;
            if constexpr (EVEN) {
                v[c] = *reinterpret_cast<const AnyVec*>(p + (j < D ? j : 0));  // (behind the row: its first, not used)
            } else if constexpr (WHOLE) {
                v[c] = *reinterpret_cast<const AnyVec*>(p + j);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) v[c][e] = j + e < D ? p[j + e] : (T)0.f;
            }
        }
        __device__ __forceinline__ void get(int t, int D, float (&x)[N]) const {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = EVEN && col(t, i) >= D ? 0.f : (float)v[i / E][i % E];
        }
    };
    // f(vector, whether it is whole) for a thread's vectors: one branch around the loads of a row's tensors, not one around
    // each
    template <class F>
    static __device__ __forceinline__ void loads(int t, int D, F&& f) {
#pragma unroll
        for (int c = 0; c < kVecs; ++c) {
            if (EVEN || (c * TPR + t) * E + E <= D) f(c, std::true_type{});
            else f(c, std::false_type{});
        }
    }
    static __device__ __forceinline__ int col(int t, int i) { return ((i / E) * TPR + t) * E + i % E; }
    static __device__ __forceinline__ void store(T* p, int t, int D, const float (&x)[N]) {
#pragma unroll
        for (int c = 0; c < kVecs; ++c) {
            const int j = (c * TPR + t) * E;
            Vec v;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = (T)x[c * E + e];
            if (j + E <= D) {
                *reinterpret_cast<AnyVec*>(p + j) = v;
            } else if constexpr (!EVEN) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (j + e < D) p[j + e] = v[e];
            }
        }
    }
    static __device__ __forceinline__ void load_f32(const float* p, int t, int D, float def, float (&x)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = col(t, i);
            x[i] = p && j < D ? p[j] : (j < D ? def : 0.f);
        }
    }
    // K sums over the row's threads, in every one of them.  Rows of more than one wave: through `red` (2 x K x 16 floats,
    // alternating halves, so one barrier a call is enough); `flip` counts the calls.
    template <int K>
    static __device__ __forceinline__ void sum(float (&v)[K], float* red, int& flip) {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = group_sum<(TPR < 64 ? TPR : 64)>(v[k]);
        if constexpr (TPR > 64) {
            float* r = red + (flip & 1) * 32;
            ++flip;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int k = 0; k < K; ++k) r[k * 16 + (threadIdx.x >> 6)] = v[k];
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k) {
                v[k] = 0.f;
#pragma unroll
                for (int w = 0; w < TPR / 64; ++w) v[k] += r[k * 16 + w];
            }
        }
    }
};

struct Args {
    const void *res, *y, *gate;
    const float *post_w, *post_b, *pre_w, *pre_b;
    int64_t n, rows_per_gate;
    int D;
    float scale, eps;
    int rms;
    void *s, *z;
    float* stats;  // (n, 4): mean and r of y, mean and r of s
    // backward
    const void *ds, *dz;
    void *dres, *dy, *dgate;
    float* part;       // (grid, 4, D): post_w, post_b, pre_w, pre_b
    float* gate_part;  // (items, D) when a gate's rows are split over items
    int64_t subs, sub_rows, items;
};

// mean and 1 / deviation of the row's values (two passes over registers)
template <class R, int kPer = R::kPer>
__device__ __forceinline__ void moments(const float (&x)[kPer], int t, int D, float eps, int rms, float* red, int& flip,
                                        float& mean, float& r) {
    mean = 0.f;
    if (!rms) {
        float v[1] = {0.f};
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[0] += x[i];
        R::template sum<1>(v, red, flip);
        mean = v[0] / (float)D;
    }
    float v[1] = {0.f};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const float c = R::col(t, i) < D ? x[i] - mean : 0.f;
        v[0] = fmaf(c, c, v[0]);
    }
    R::template sum<1>(v, red, flip);
    r = 1.f / sqrtf(v[0] / (float)D + eps);
}

template <class T, class R>
__global__ __launch_bounds__(R::kThreads) void fwd_kernel(Args a) {
    constexpr int kPer = R::kPer;
    __shared__ float red[64];
    int flip = 0;
    const int t = threadIdx.x % R::TPRv, slot = R::kSlots > 1 ? threadIdx.x / R::TPRv : 0, D = a.D;
    float pw[kPer], pb[kPer], qw[kPer], qb[kPer];
    R::load_f32(a.post_w, t, D, 1.f, pw);
    R::load_f32(a.post_b, t, D, 0.f, pb);
    R::load_f32(a.pre_w, t, D, 1.f, qw);
    R::load_f32(a.pre_b, t, D, 0.f, qb);
    typename R::Raw raw_y, raw_s, raw_g;
    const int64_t step = (int64_t)gridDim.x * R::kSlots;
    auto fetch = [&](int64_t base) {  // the row that this thread's slot has from `base` on
        const int64_t row = min(base + slot, a.n - 1);
        const T* g = (const T*)a.gate + (a.gate ? row / a.rows_per_gate * D : 0);
        R::loads(t, D, [&](int c, auto whole) {
            constexpr bool W = decltype(whole)::value;
            raw_y.template load<W>((const T*)a.y + row * D, t, D, c);
            raw_s.template load<W>((const T*)a.res + row * D, t, D, c);
            if (a.gate) raw_g.template load<W>(g, t, D, c);
        });
    };
    // (every thread of a workgroup makes the same number of turns: the row sums may hold a barrier)
    int64_t base = (int64_t)blockIdx.x * R::kSlots;
    if (base < a.n) fetch(base);
    for (; base < a.n; base += step) {
        const int64_t row = base + slot;
        const bool live = row < a.n;
        float x[kPer], s[kPer], g[kPer], m, r;
        raw_y.get(t, D, x);
        raw_s.get(t, D, s);
        if (a.gate) raw_g.get(t, D, g);
        if (base + step < a.n) fetch(base + step);  // the next row is on its way during this one's sums
        moments<R>(x, t, D, a.eps, a.rms, red, flip, m, r);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float b = fmaf((x[i] - m) * r, pw[i], pb[i]);
            s[i] = a.gate ? fmaf(g[i], b, a.scale * s[i]) : fmaf(a.scale, s[i], b);
            if (R::col(t, i) >= D) s[i] = 0.f;
        }
        if (live) R::store((T*)a.s + row * D, t, D, s);
        float m2 = 0.f, r2 = 0.f;
        if (a.pre_w) {
            moments<R>(s, t, D, a.eps, a.rms, red, flip, m2, r2);
#pragma unroll
            for (int i = 0; i < kPer; ++i) s[i] = fmaf((s[i] - m2) * r2, qw[i], qb[i]);
            if (live) R::store((T*)a.z + row * D, t, D, s);
        }
        if (live && t == 0) *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(m, r, m2, r2);
    }
}

// the workgroup's column sums of one accumulator over its row slots -> out[0..D)
template <class R, class Put, int kPer = R::kPer>
__device__ __forceinline__ void column_sums(const float (&acc)[kPer], int t, int slot, int D, float* buf, Put&& put) {
    if constexpr (R::kSlots == 1) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (R::col(t, i) < D) put(R::col(t, i), acc[i]);
    } else {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; ++i) buf[(slot * R::TPRv + t) * kPer + i] = acc[i];
        __syncthreads();
        // buf[slot][thread][value]: one (thread, value) pair per column
        for (int c = threadIdx.x; c < R::TPRv * kPer; c += R::kThreads) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < R::kSlots; ++k) v += buf[k * R::TPRv * kPer + c];
            const int j = R::col(c / kPer, c % kPer);
            if (j < D) put(j, v);
        }
    }
}

// GATE: 0 none, 1 a row of its own for every row (dgate written at once), 2 shared by rows_per_gate rows.
// Items: rows_per_gate rows (all rows without a shared gate) in `subs` pieces of sub_rows; a workgroup takes items
// blockIdx.x, + gridDim.x, ...: a shared gate's sums are closed at the end of each item, the weights' at the end of all.
template <class T, class R, int GATE>
__global__ __launch_bounds__(R::kThreads) void bwd_kernel(Args a) {
    constexpr int kPer = R::kPer;
    __shared__ float red[64];
    __shared__ float buf[R::kSlots > 1 ? R::kThreads * kPer : 1];
    int flip = 0;
    const int t = threadIdx.x % R::TPRv, slot = R::kSlots > 1 ? threadIdx.x / R::TPRv : 0, D = a.D;
    const float inv_d = 1.f / (float)D, centre = a.rms ? 0.f : 1.f;
    float pw[kPer], pb[kPer], qw[kPer];
    R::load_f32(a.post_w, t, D, 1.f, pw);
    R::load_f32(a.post_b, t, D, 0.f, pb);
    R::load_f32(a.pre_w, t, D, 1.f, qw);
    float acc[4][R::kLean ? 1 : kPer], gacc[kPer];
    __shared__ floatx4 far[R::kLean ? 4 * kPer / 4 * R::kThreads : 1];  // (a thread's own columns: no barrier)
    // the sums k = 0 .. 3 of the thread's columns: f(i, so far) is the new one of value i
    auto add = [&](int k, auto f) {
        if constexpr (R::kLean) {
#pragma unroll
            for (int c = 0; c < kPer / 4; ++c) {
                floatx4& p = far[(k * (kPer / 4) + c) * R::kThreads + threadIdx.x];
                floatx4 v = p;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = f(4 * c + e, v[e]);
                p = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) acc[k][i] = f(i, acc[k][i]);
        }
    };
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (R::kLean) {
            for (int c = 0; c < kPer / 4; ++c)
                far[(k * (kPer / 4) + c) * R::kThreads + threadIdx.x] = floatx4{0.f, 0.f, 0.f, 0.f};
        } else {
            for (int i = 0; i < kPer; ++i) acc[k][i] = 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) gacc[i] = 0.f;
    typename R::Raw raw_y, raw_s, raw_d, raw_z, raw_g;
    float4 next_st;
    // this thread's slot of the rows from `base` on (the last one again behind `end`)
    auto fetch = [&](int64_t base, int64_t end, int64_t group) {
        const int64_t row = min(base + slot, end - 1);
        next_st = *reinterpret_cast<const float4*>(a.stats + row * 4);
        R::loads(t, D, [&](int c, auto whole) {
            constexpr bool W = decltype(whole)::value;
            raw_y.template load<W>((const T*)a.y + row * D, t, D, c);
            raw_s.template load<W>((const T*)a.res + row * D, t, D, c);
            if (GATE) raw_g.template load<W>((const T*)a.gate + (GATE == 1 ? row : group) * D, t, D, c);
            if (a.ds) raw_d.template load<W>((const T*)a.ds + row * D, t, D, c);
            if (a.dz) raw_z.template load<W>((const T*)a.dz + row * D, t, D, c);
        });
    };
    for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
        const int64_t group = item / a.subs, first = (item % a.subs) * a.sub_rows;
        const int64_t begin = group * a.rows_per_gate + first;
        const int64_t end = group * a.rows_per_gate + min(a.rows_per_gate, first + a.sub_rows);
        if (!R::kLean) fetch(begin, end, group);
        for (int64_t base = begin; base < end; base += R::kSlots) {
            const bool live = base + slot < end;
            const int64_t row = live ? base + slot : end - 1;
            if (R::kLean) fetch(base, end, group);
            const float4 st = next_st;
            float y[kPer], s[kPer], d[kPer], g[kPer], dz[kPer];
            raw_y.get(t, D, y);
            raw_s.get(t, D, s);
            if (a.ds) raw_d.get(t, D, d);
            if (a.dz) raw_z.get(t, D, dz);
            if (GATE) raw_g.get(t, D, g);
            if (!R::kLean && base + R::kSlots < end) fetch(base + R::kSlots, end, group);  // on its way during this row's sums
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (!live || !a.ds) d[i] = 0.f;
                const bool in = R::col(t, i) < D;
                y[i] = in ? (y[i] - st.x) * st.y : 0.f;
                const float br = fmaf(y[i], pw[i], pb[i]);
                s[i] = GATE ? fmaf(g[i], br, a.scale * s[i]) : fmaf(a.scale, s[i], br);
                s[i] = in ? (s[i] - st.z) * st.w : 0.f;
            }
            if (a.dz) {
                float v[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    if (!live) dz[i] = 0.f;
                }
                add(2, [&](int i, float v) { return fmaf(dz[i], s[i], v); });
                add(3, [&](int i, float v) { return v + dz[i]; });
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    dz[i] *= qw[i];
                    v[0] = fmaf(dz[i], s[i], v[0]);
                    v[1] += dz[i];
                }
                R::template sum<2>(v, red, flip);
                v[0] *= inv_d;
                v[1] *= inv_d * centre;
#pragma unroll
                for (int i = 0; i < kPer; ++i) d[i] = fmaf(dz[i] - fmaf(s[i], v[0], v[1]), st.w, d[i]);
            }
            if (a.dres && live) {
                float o[kPer];
#pragma unroll
                for (int i = 0; i < kPer; ++i) o[i] = a.scale * d[i];
                R::store((T*)a.dres + row * D, t, D, o);
            }
            if (GATE == 1 && a.dgate && live) {
                float o[kPer];
#pragma unroll
                for (int i = 0; i < kPer; ++i) o[i] = d[i] * fmaf(y[i], pw[i], pb[i]);
                R::store((T*)a.dgate + row * D, t, D, o);
            }
            float v[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (R::col(t, i) >= D) d[i] = 0.f;
                if (GATE == 2) gacc[i] = fmaf(d[i], fmaf(y[i], pw[i], pb[i]), gacc[i]);
                if (GATE) d[i] *= g[i];
            }
            add(0, [&](int i, float v) { return fmaf(d[i], y[i], v); });
            add(1, [&](int i, float v) { return v + d[i]; });
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                d[i] *= pw[i];
                v[0] = fmaf(d[i], y[i], v[0]);
                v[1] += d[i];
            }
            if (a.dy) {
                R::template sum<2>(v, red, flip);
                v[0] *= inv_d;
                v[1] *= inv_d * centre;
#pragma unroll
                for (int i = 0; i < kPer; ++i) d[i] = (d[i] - fmaf(y[i], v[0], v[1])) * st.y;
                if (live) R::store((T*)a.dy + row * D, t, D, d);
            }
        }
        if (GATE == 2 && a.dgate) {
            if (a.subs == 1)
                column_sums<R>(gacc, t, slot, D, buf,
                               [&](int j, float v) { Elem<T>::put((T*)a.dgate + group * D + j, v); });
            else
                column_sums<R>(gacc, t, slot, D, buf, [&](int j, float v) { a.gate_part[item * D + j] = v; });
#pragma unroll
            for (int i = 0; i < kPer; ++i) gacc[i] = 0.f;
        }
    }
    if (a.part)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                v[i] = R::kLean ? far[(k * (kPer / 4) + i / 4) * R::kThreads + threadIdx.x][i % 4] : acc[k][R::kLean ? 0 : i];
            column_sums<R>(v, t, slot, D, buf,
                           [&](int j, float x) { a.part[((int64_t)blockIdx.x * 4 + k) * D + j] = x; });
        }
}

// out[g][j] = sum over m < rows of part[g * rows + m][j], j < width: 16 columns x 64 row lanes a workgroup, then the
// lanes' sums in order (64 columns x 16 lanes took 13 us for 1024 rows of 512: one load after another)
constexpr int kCols = 16;
template <class T>
__global__ __launch_bounds__(1024) void column_reduce_kernel(const float* __restrict__ part, int64_t rows, int64_t width,
                                                             int64_t col_groups, T* __restrict__ out) {
    __shared__ float buf[64][kCols + 1];
    const int64_t g = blockIdx.x / col_groups, j = blockIdx.x % col_groups * kCols + threadIdx.x % kCols;
    const int lane = threadIdx.x / kCols;
    float v = 0.f;
    if (j < width) {
        const float* p = part + g * rows * width + j;
#pragma unroll 8
        for (int64_t m = lane; m < rows; m += 64) v += p[m * width];
    }
    buf[lane][threadIdx.x % kCols] = v;
    __syncthreads();
    if (threadIdx.x < 4 * kCols) {  // a quarter of the lanes each, then the quarters
        const int c = threadIdx.x % kCols, q = threadIdx.x / kCols;
        v = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) v += buf[16 * q + k][c];
        v += __shfl_xor(v, 16, 64);
        v += __shfl_xor(v, 32, 64);
        if (q == 0 && j < width) Elem<T>::put(out + g * width + j, v);
    }
}

// f(Row<...>{}) for a checked dim: the fewest threads a row (at least 16) that hold it at one 16-byte vector each, 8
// values beyond 4096
template <class T, class F>
void with_row(int64_t D, bool even, F&& f) {
    constexpr int N = Elem<T>::V;
    auto pick = [&](auto even) {
        constexpr bool EVEN = decltype(even)::value;
        if (D <= 16 * N) f(Row<T, 16, N, EVEN>{});
        else if (D <= 32 * N) f(Row<T, 32, N, EVEN>{});
        else if (D <= 64 * N) f(Row<T, 64, N, EVEN>{});
        else if (D <= 128 * N) f(Row<T, 128, N, EVEN>{});
        else if (D <= 256 * N) f(Row<T, 256, N, EVEN>{});
        else if (EVEN || D <= 512 * N) f(Row<T, 512, N, EVEN>{});
        else {
            if constexpr (N == 4) {
                if (D <= 4096) return f(Row<T, 1024, 4, false>{});
            }
            f(Row<T, 1024, 8, false>{});
        }
    };
    if (even && D % N == 0 && D <= 512 * N) pick(std::true_type{});
    else pick(std::false_type{});
}

// workgroups of a layout that fill the chip: 16 waves on each of 256 CUs, at most 1024 (their partial rows are written)
constexpr int64_t fill_of(int64_t threads) { return std::min<int64_t>(1024, 256 * 1024 / threads); }
template <class R>
constexpr int64_t fill() {
    return fill_of(R::kThreads);
}
// the most of them that any layout of a dim takes (at most 8 values a thread)
int64_t most_groups(int64_t D) { return D <= 2048 ? 1024 : D <= 4096 ? fill_of(512) : fill_of(1024); }

struct Plan {
    int64_t subs, sub_rows, items, grid;
};
// pieces of the backward: the rows of a shared gate (else all rows) cut so that there are enough items to fill the chip,
// each a whole number of turns; the grid (and with it the partial rows) is at most what runs at once
Plan plan(int64_t n, int64_t rows_per_gate, int64_t slots, int64_t fill) {
    const int64_t groups = n / rows_per_gate;
    Plan p;
    const int64_t turns = (rows_per_gate + slots - 1) / slots;
    int64_t subs = std::min(turns, std::max<int64_t>(1, fill / groups));
    p.sub_rows = (turns + subs - 1) / subs * slots;
    p.subs = (rows_per_gate + p.sub_rows - 1) / p.sub_rows;
    p.items = groups * p.subs;
    p.grid = std::min(p.items, fill);
    return p;
}

bool sizes_ok(int64_t n, int64_t D, int64_t rows_per_gate) {
    return n >= 1 && D >= 1 && D <= kMaxDim && n <= (1ll << 40) / D && rows_per_gate >= 1 && rows_per_gate <= n &&
           n % rows_per_gate == 0;
}

}  // namespace

ASME_API int asme_gated_residual_norm_fwd(const void* res, const void* y, const void* gate, int64_t rows_per_gate,
                                          const float* post_w, const float* post_b, const float* pre_w,
                                          const float* pre_b, int64_t n, int64_t dim, float residual_scale, float eps,
                                          int rms, int dtype, void* s_out, void* z_out, float* stats, void* stream) {
    ASME_CHECK_ARG(res && y && post_w && s_out && stats, "asme_gated_residual_norm_fwd: null pointer");
    ASME_CHECK_ARG(!pre_w || z_out, "asme_gated_residual_norm_fwd: z_out missing");
    ASME_CHECK_ARG(dtype_ok(dtype), "asme_gated_residual_norm_fwd: dtype is 0 (fp32) or 1 (bf16)");
    ASME_CHECK_ARG(sizes_ok(n, dim, gate ? rows_per_gate : 1), "asme_gated_residual_norm_fwd: bad size");
    ASME_CHECK_ARG(eps >= 0.f, "asme_gated_residual_norm_fwd: eps >= 0");
    Args a{};
    a.res = res, a.y = y, a.gate = gate, a.post_w = post_w, a.post_b = post_b, a.pre_w = pre_w, a.pre_b = pre_b;
    a.n = n, a.rows_per_gate = gate ? rows_per_gate : 1, a.D = (int)dim, a.scale = residual_scale, a.eps = eps;
    a.rms = rms, a.s = s_out, a.z = z_out, a.stats = stats;
    with_dtype(dtype, [&](auto e) {
        using T = decltype(e);
        with_row<T>(dim, aligned({res, y, gate, s_out, z_out}), [&](auto r) {
            using R = decltype(r);
            const int64_t turns = (n + R::kSlots - 1) / R::kSlots;
            hipLaunchKernelGGL((fwd_kernel<T, R>), dim3((unsigned)std::min(turns, 2 * fill<R>())),
                               dim3(R::kThreads), 0, (hipStream_t)stream, a);
        });
    });
    ASME_LAUNCH_CHECK("asme_gated_residual_norm_fwd");
}

// bytes, whatever the layout that the call takes; 0 for sizes that the calls refuse
ASME_API int64_t asme_gated_residual_norm_bwd_workspace(int64_t n, int64_t dim, int64_t rows_per_gate) {
    if (!sizes_ok(n, dim, rows_per_gate)) return 0;
    // partial rows of the weights, and (only where a gate's rows are cut into pieces: then no more pieces than workgroups)
    // of the gate
    return std::min(n, most_groups(dim)) * 5 * dim * 4;
}

// rows_per_gate: as in the forward; n (all rows) without a gate or with a gate row for every row (gate_rows = 1)
ASME_API int asme_gated_residual_norm_bwd(const void* res, const void* y, const void* gate, int64_t rows_per_gate,
                                          const float* post_w, const float* post_b, const float* pre_w, int64_t n,
                                          int64_t dim, float residual_scale, int rms, int dtype, const float* stats,
                                          const void* ds, const void* dz, void* dres, void* dy, void* dgate,
                                          float* dw, void* workspace, int64_t ws_bytes, void* stream) {
    ASME_CHECK_ARG(res && y && post_w && stats && workspace, "asme_gated_residual_norm_bwd: null pointer");
    ASME_CHECK_ARG(!dz || pre_w, "asme_gated_residual_norm_bwd: dz without the norm's weight");
    ASME_CHECK_ARG(!dgate || gate, "asme_gated_residual_norm_bwd: dgate without a gate");
    ASME_CHECK_ARG(dtype_ok(dtype), "asme_gated_residual_norm_bwd: dtype is 0 (fp32) or 1 (bf16)");
    ASME_CHECK_ARG(sizes_ok(n, dim, gate ? rows_per_gate : 1), "asme_gated_residual_norm_bwd: bad size");
    const bool shared = gate && rows_per_gate > 1;
    const int64_t rows = shared ? rows_per_gate : n;
    ASME_CHECK_ARG(ws_bytes >= asme_gated_residual_norm_bwd_workspace(n, dim, rows),
                   "asme_gated_residual_norm_bwd: workspace too small");
    Args a{};
    a.res = res, a.y = y, a.gate = gate, a.post_w = post_w, a.post_b = post_b, a.pre_w = pre_w;
    a.n = n, a.rows_per_gate = rows, a.D = (int)dim, a.scale = residual_scale, a.rms = rms;
    a.stats = const_cast<float*>(stats), a.ds = ds, a.dz = dz, a.dres = dres, a.dy = dy, a.dgate = dgate;
    a.part = dw ? (float*)workspace : nullptr;
    hipStream_t st = (hipStream_t)stream;
    const unsigned cg = (unsigned)((dim + kCols - 1) / kCols), cg4 = (unsigned)((4 * dim + kCols - 1) / kCols);
    Plan p{};
    with_dtype(dtype, [&](auto e) {
        using T = decltype(e);
        with_row<T>(dim, aligned({res, y, gate, ds, dz, dres, dy, dgate}), [&](auto r) {
            using R = decltype(r);
            p = plan(n, rows, R::kSlots, fill<R>());
            a.gate_part = (float*)workspace + p.grid * 4 * dim;
            a.subs = p.subs, a.sub_rows = p.sub_rows, a.items = p.items;
            const dim3 grid((unsigned)p.grid), block(R::kThreads);
            if (!gate) hipLaunchKernelGGL((bwd_kernel<T, R, 0>), grid, block, 0, st, a);
            else if (!shared) hipLaunchKernelGGL((bwd_kernel<T, R, 1>), grid, block, 0, st, a);
            else hipLaunchKernelGGL((bwd_kernel<T, R, 2>), grid, block, 0, st, a);
        });
        if (shared && dgate && p.subs > 1)
            hipLaunchKernelGGL(column_reduce_kernel<T>, dim3((unsigned)(p.items / p.subs) * cg), dim3(1024), 0, st,
                               a.gate_part, p.subs, dim, (int64_t)cg, (T*)dgate);
    });
    if (dw)
        hipLaunchKernelGGL(column_reduce_kernel<float>, dim3(cg4), dim3(1024), 0, st, a.part, p.grid, 4 * dim,
                           (int64_t)cg4, dw);
    ASME_LAUNCH_CHECK("asme_gated_residual_norm_bwd");
}
