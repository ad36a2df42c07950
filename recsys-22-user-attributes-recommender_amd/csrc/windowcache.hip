// Serving sliding-window attention with sinks (window.hip): the ring cache of a sequence's visible keys and values, and
// the attention of one new token against it.
//
// The cache of a sequence holds sinks + window slots.  Position p lives in slot p while p < sinks and in slot
// sinks + (p - sinks) mod window after that, so once position n is stored the slots hold exactly what position n sees:
// the sinks and the last `window` positions, in min(n + 1, slots) slots.  A softmax does not depend on the order of its
// terms: no mask and no position is needed, and memory stays bounded for a history of any length.
//
// step: out[b][h] = sum_j softmax_j(scale q[b][h] . K_j) V_j over the held slots, K and V of the new token among them;
// the new token is stored in the same pass.  Bound by reading the cache once.  A row of D values is read by D / V lanes
// (V = values of a 16-byte vector), so a wave reads 64 V / D rows of 1 KiB in one instruction; each lane group runs its
// own softmax (maximum, sum, weighted values) over its rows for the query heads that share the key head, kRows rows a
// turn, and the groups, waves and -- where there are few sequences -- workgroups along the slots are merged at the end
// in a fixed order.  Scores, statistics and sums are fp32; the output is rounded once.
// Measured: 64 sequences, 32 heads on 8, D = 128, 4100 slots, bf16: 215 us for 1023 MB, 4.7 TB/s, what a copy reaches; one
// sequence of two heads, 130 slots of 64 fp32: 3.6 us of 14 that the call takes.
// fill: bound by latency and the copy (8 prompts of up to 2000, D = 64, bf16: 4 us).
#include "elem.h"

using namespace asme;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256;
constexpr int kRows = 4;         // rows of a lane group per turn
constexpr int kMaxSplits = 64;   // one lane of the merging wave each
constexpr int kMaxShared = 8;    // query heads of a key head per workgroup

int64_t step_splits(int64_t heads, int64_t slots) {  // heads: workgroups that the sequences' key heads make already
    const int64_t want = (1024 + heads - 1) / heads, most = (slots + 255) / 256;
    return std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxSplits}));
}

struct StepArgs {
    const void *q, *k, *v;
    void *cache_k, *cache_v, *out;
    const int64_t* lengths;
    int64_t slots, sinks, per_split;
    int kv_heads, group, chunks, splits;
    float scale;  // of the scores, in base 2
    float* part;  // (batch * heads, splits, D + 2): weighted values, maximum, sum
};

template <class T, int D, int G>
__global__ __launch_bounds__(kThreads) void step_kernel(StepArgs a) {
    constexpr int V = Elem<T>::V, LPR = D / V, NG = kThreads / LPR;  // lanes a row, lane groups
    const int split = blockIdx.x % a.splits, chunk = blockIdx.x / a.splits % a.chunks;
    const int64_t bk = blockIdx.x / a.splits / a.chunks;  // sequence and key head
    const int64_t b = bk / a.kv_heads;
    const int kh = (int)(bk % a.kv_heads), heads = a.kv_heads * a.group;
    const int h0 = kh * a.group + chunk * kMaxShared, nh = min(G, a.group - chunk * kMaxShared);
    const int lane = threadIdx.x & 63, sub = lane % LPR, gid = threadIdx.x / LPR;
    const int64_t len = a.lengths[b];
    T* out = (T*)a.out + (b * heads + h0) * D;
    if (len < 0) {  // a sequence that takes no step
        if (split == 0)
            for (int i = threadIdx.x; i < nh * D; i += kThreads) Elem<T>::put(out + i, 0.f);
        if (a.splits > 1)
            for (int i = threadIdx.x; i < nh * (D + 2); i += kThreads)
                a.part[((b * heads + h0 + i / (D + 2)) * a.splits + split) * (D + 2) + i % (D + 2)] = 0.f;
        return;
    }
    const int64_t window = a.slots - a.sinks;
    const int64_t to = len < a.sinks ? len : a.sinks + (len - a.sinks) % window;
    const int64_t held = min(len + 1, a.slots);
    const int64_t begin = split * a.per_split, end = min(held, begin + a.per_split);
    T* ck = (T*)a.cache_k + bk * a.slots * D;
    T* cv = (T*)a.cache_v + bk * a.slots * D;
    const T* nk = (const T*)a.k + bk * D;
    const T* nv = (const T*)a.v + bk * D;
    float q[G][V], acc[G][V], m[G], l[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        m[g] = -INFINITY, l[g] = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) q[g][i] = acc[g][i] = 0.f;
        if (g < nh) Elem<T>::load((const T*)a.q + (b * heads + h0 + g) * D + sub * V, q[g]);
    }
    for (int64_t r0 = begin + gid; r0 < end; r0 += NG * kRows) {
        float kk[kRows][V], vv[kRows][V], s[kRows][G];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            const int64_t r = min(r0 + u * NG, end - 1);
            Elem<T>::load((r == to ? nk : ck + r * D) + sub * V, kk[u]);
            Elem<T>::load((r == to ? nv : cv + r * D) + sub * V, vv[u]);
        }
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            if (r0 + u * NG == to && to < end && chunk == 0) {  // (behind `end` the row is another workgroup's)
                Elem<T>::store(ck + to * D + sub * V, kk[u]);
                Elem<T>::store(cv + to * D + sub * V, vv[u]);
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float x = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) x = fmaf(kk[u][i], q[g][i], x);
                x = group_sum<LPR>(x) * a.scale;
                s[u][g] = r0 + u * NG < end ? x : -INFINITY;
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float t = s[0][g];
#pragma unroll
            for (int u = 1; u < kRows; ++u) t = fmaxf(t, s[u][g]);
            if (t > m[g]) {
                const float f = __builtin_amdgcn_exp2f(m[g] - t);
                l[g] *= f;
#pragma unroll
                for (int i = 0; i < V; ++i) acc[g][i] *= f;
                m[g] = t;
            }
#pragma unroll
            for (int u = 0; u < kRows; ++u) {
                const float p = __builtin_amdgcn_exp2f(s[u][g] - m[g]);
                l[g] += p;
#pragma unroll
                for (int i = 0; i < V; ++i) acc[g][i] = fmaf(p, vv[u][i], acc[g][i]);
            }
        }
    }
    // the lane groups of a wave, then the waves
    __shared__ float part[kThreads / 64][G][D + 2];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        float M = m[g];
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
        const float f = m[g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[g] - M);
        l[g] *= f;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[g][i] *= f;
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1) {
            l[g] += __shfl_xor(l[g], o, 64);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[g][i] += __shfl_xor(acc[g][i], o, 64);
        }
        if (lane < LPR) {
            float* p = part[threadIdx.x >> 6][g];
#pragma unroll
            for (int i = 0; i < V; ++i) p[lane * V + i] = acc[g][i];
            if (lane == 0) p[D] = M, p[D + 1] = l[g];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * D; i += kThreads) {
        const int g = i / D, c = i % D;
        float M = part[0][g][D], L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 1; w < kThreads / 64; ++w) M = fmaxf(M, part[w][g][D]);
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) {
            const float f = part[w][g][D] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(part[w][g][D] - M);
            L = fmaf(part[w][g][D + 1], f, L);
            o = fmaf(part[w][g][c], f, o);
        }
        if (a.splits == 1) {
            Elem<T>::put(out + i, o / L);
        } else {
            float* p = a.part + ((b * heads + h0 + g) * a.splits + split) * (D + 2);
            p[c] = o;
            if (c == 0) p[D] = M, p[D + 1] = L;
        }
    }
}

// one wave per (sequence, head): lane s holds split s's state, then lane c the output columns c, c + 64
template <class T, int D>
__global__ __launch_bounds__(256) void merge_kernel(const float* __restrict__ part, int64_t n, int splits,
                                                    T* __restrict__ out) {
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= n) return;
    const int lane = threadIdx.x & 63;
    const float* p = part + r * splits * (D + 2);
    float m = -INFINITY, l = 0.f;
    if (lane < splits) m = p[lane * (D + 2) + D], l = p[lane * (D + 2) + D + 1];
    const float M = wave_max(l != 0.f ? m : -INFINITY);  // (an empty split: l = 0; a NaN goes on)
    const float f = l != 0.f ? __builtin_amdgcn_exp2f(m - M) : 0.f;
    const float L = wave_sum(l * f);
    for (int c = lane; c < D + (64 - D % 64) % 64; c += 64) {
        float o = 0.f;
        for (int s = 0; s < splits; ++s) o = fmaf(c < D ? p[s * (D + 2) + c] : 0.f, __shfl(f, s, 64), o);
        if (c < D) Elem<T>::put(out + r * D + c, L != 0.f ? o / L : o);
    }
}

// the slots of a fresh cache that a prompt's positions fall on: one 16-byte vector of K and V a thread
template <class T>
__global__ __launch_bounds__(256) void fill_kernel(const T* __restrict__ k, const T* __restrict__ v, int64_t kb, int64_t kt,
                                                   int64_t kh, int64_t vb, int64_t vt, int64_t vh,
                                                   const int64_t* __restrict__ lengths, int64_t seq_len, int64_t total,
                                                   int kv_heads, int D, int64_t slots, int64_t sinks,
                                                   T* __restrict__ cache_k, T* __restrict__ cache_v) {
    constexpr int V = Elem<T>::V;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int vecs = D / V, c = (int)(i % vecs) * V;
    const int64_t slot = i / vecs % slots, bh = i / vecs / slots, b = bh / kv_heads, h = bh % kv_heads;
    const int64_t last = min(lengths[b], seq_len) - 1;
    int64_t at = slot;
    if (slot >= sinks) {
        if (last < slot) return;  // nothing has come to this slot yet
        at = last - (last - slot) % (slots - sinks);
    }
    if (at > last) return;
    float x[V];
    Elem<T>::load(k + b * kb + at * kt + h * kh + c, x);
    Elem<T>::store(cache_k + (bh * slots + slot) * D + c, x);
    Elem<T>::load(v + b * vb + at * vt + h * vh + c, x);
    Elem<T>::store(cache_v + (bh * slots + slot) * D + c, x);
}

bool dim_ok(int64_t D) { return D == 16 || D == 32 || D == 64 || D == 128; }
bool sizes_ok(int64_t batch, int64_t heads, int64_t kv_heads, int64_t D, int64_t slots, int64_t sinks) {
    return batch >= 1 && kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && dim_ok(D) && sinks >= 0 &&
           slots > sinks && heads <= 65536 && batch <= (1ll << 24) && batch * heads <= (1ll << 24) &&
           slots <= (1ll << 40) / (batch * kv_heads * D);
}
template <class F>
void with_dim(int64_t D, F&& f) {
    if (D == 16) f(std::integral_constant<int, 16>{});
    else if (D == 32) f(std::integral_constant<int, 32>{});
    else if (D == 64) f(std::integral_constant<int, 64>{});
    else f(std::integral_constant<int, 128>{});
}

}  // namespace

// bytes (0 where one workgroup a key head is enough, and for sizes that the call refuses)
ASME_API int64_t asme_window_step_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                            int64_t slots) {
    if (!sizes_ok(batch, heads, kv_heads, head_dim, slots, 0)) return 0;
    const int64_t splits = step_splits(batch * kv_heads, slots);
    return splits == 1 ? 0 : batch * heads * splits * (head_dim + 2) * 4;
}

ASME_API int asme_window_step(const void* q, const void* k, const void* v, void* cache_k, void* cache_v,
                              const int64_t* lengths, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                              int64_t slots, int64_t sinks, float scale, int dtype, void* workspace, int64_t ws_bytes,
                              void* out, void* stream) {
    ASME_CHECK_ARG(q && k && v && cache_k && cache_v && lengths && out, "asme_window_step: null pointer");
    ASME_CHECK_ARG(dtype_ok(dtype), "asme_window_step: dtype is 0 (fp32) or 1 (bf16)");
    ASME_CHECK_ARG(sizes_ok(batch, heads, kv_heads, head_dim, slots, sinks), "asme_window_step: bad size");
    ASME_CHECK_ARG(scale > 0.f && scale < INFINITY, "asme_window_step: scale > 0");
    ASME_CHECK_ARG(aligned({q, k, v, cache_k, cache_v, out}), "asme_window_step: 16-byte alignment");
    ASME_CHECK_ARG(ws_bytes >= asme_window_step_workspace(batch, heads, kv_heads, head_dim, slots),
                   "asme_window_step: workspace too small");
    const int64_t splits = step_splits(batch * kv_heads, slots), group = heads / kv_heads;
    ASME_CHECK_ARG(splits == 1 || workspace, "asme_window_step: null workspace");
    StepArgs a{q, k, v, cache_k, cache_v, out, lengths, slots, sinks, (slots + splits - 1) / splits, (int)kv_heads,
               (int)group, (int)((group + kMaxShared - 1) / kMaxShared), (int)splits, scale * kLog2e, (float*)workspace};
    const dim3 grid((unsigned)(batch * kv_heads * a.chunks * splits)), block(kThreads);
    hipStream_t s = (hipStream_t)stream;
    with_dtype(dtype, [&](auto e) {
        using T = decltype(e);
        with_dim(head_dim, [&](auto dim) {
            constexpr int D = decltype(dim)::value;
            if (group == 1) hipLaunchKernelGGL((step_kernel<T, D, 1>), grid, block, 0, s, a);
            else if (group == 2) hipLaunchKernelGGL((step_kernel<T, D, 2>), grid, block, 0, s, a);
            else if (group <= 4) hipLaunchKernelGGL((step_kernel<T, D, 4>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((step_kernel<T, D, kMaxShared>), grid, block, 0, s, a);
            if (splits > 1)
                hipLaunchKernelGGL((merge_kernel<T, D>), dim3((unsigned)((batch * heads + 3) / 4)), dim3(256), 0, s,
                                   a.part, batch * heads, (int)splits, (T*)out);
        });
    });
    ASME_LAUNCH_CHECK("asme_window_step");
}

ASME_API int asme_window_cache_fill(const void* k, const void* v, int64_t k_batch, int64_t k_token, int64_t k_head,
                                    int64_t v_batch, int64_t v_token, int64_t v_head, const int64_t* lengths,
                                    int64_t batch, int64_t seq_len, int64_t kv_heads, int64_t head_dim, int64_t slots,
                                    int64_t sinks, int dtype, void* cache_k, void* cache_v, void* stream) {
    ASME_CHECK_ARG(k && v && lengths && cache_k && cache_v, "asme_window_cache_fill: null pointer");
    ASME_CHECK_ARG(dtype_ok(dtype), "asme_window_cache_fill: dtype is 0 (fp32) or 1 (bf16)");
    ASME_CHECK_ARG(seq_len >= 1 && sizes_ok(batch, kv_heads, kv_heads, head_dim, slots, sinks),
                   "asme_window_cache_fill: bad size");
    const int64_t V = 16 / dtype_size(dtype);
    ASME_CHECK_ARG(aligned({k, v, cache_k, cache_v}) && k_batch % V == 0 && k_token % V == 0 && k_head % V == 0 &&
                       v_batch % V == 0 && v_token % V == 0 && v_head % V == 0,
                   "asme_window_cache_fill: 16-byte alignment");
    const int64_t total = batch * kv_heads * slots * (head_dim / V);
    ASME_CHECK_ARG((total + 255) / 256 < (1ll << 31), "asme_window_cache_fill: bad size");
    with_dtype(dtype, [&](auto e) {
        using T = decltype(e);
        hipLaunchKernelGGL(fill_kernel<T>, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                           (const T*)k, (const T*)v, k_batch, k_token, k_head, v_batch, v_token, v_head, lengths, seq_len,
                           total, (int)kv_heads, (int)head_dim, slots, sinks, (T*)cache_k, (T*)cache_v);
    });
    ASME_LAUNCH_CHECK("asme_window_cache_fill");
}
