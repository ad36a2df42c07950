// Sliding-window attention with sinks, forward and backward, next to the full masked attention (attention.hip): every
// query sees the last `window` positions up to its own (or `window` - 1 on both sides) and, however far back, the first
// `sinks` positions -- a user's attributes in front of a long history.
//
//   S = scale Q K^T over the visible pairs, P = softmax(S), O = P V
//   visible(i, j): valid i and j, and  causal: 0 <= i - j < window or j <= i, j < sinks
//                                      else:   |i - j| < window    or j < sinks
//   D_i = dO_i . O_i;  dP = dO V^T;  dS = P (dP - D);  dQ = scale dS K;  dV = P^T dO;  dK = scale dS^T Q
// (dK, dV summed over the query heads that share a key head).  A position that is not valid is neither query nor key:
// what it holds is not read into any product, its rows of O, dQ, dK and dV are 0.
//
// Every pass is one skeleton over a pair of stationary and streamed rows:
//   stationary  32 rows a wave as MFMA B fragments in registers for the whole kernel
//   streamed    64-row tiles of two tensors through LDS, the next tile on its way in registers during this one's products
//   X = A_streamed . B_stationary^T (32x32x16): lane (stationary row c, half h) holds streamed rows 8 (i >> 2) + 4 h +
//   (i & 3), which are -- as pairs of registers converted to bf16 -- the B fragment of the product that sums over the
//   streamed rows: Y^T[f][c] += streamed^T[f][rows] . P[rows][c], the streamed tile read back transposed
//   (ds_read_b64_tr_b16).  No lane moves a value, except for the row maximum's two halves.
//     forward   stationary Q         streamed K, V:  S -> P -> O^T += V^T P^T, online softmax
//     dQ        stationary Q, dO     streamed K, V:  S, dP -> dS -> dQ^T += K^T dS^T; writes D for the next pass
//     dK, dV    stationary K, V      streamed Q, dO: S, dP -> P, dS -> dV^T += dO^T P, dK^T += Q^T dS
// Tiles outside every row's window are not visited, 32x32 blocks outside this wave's are skipped, and only blocks on a
// border (diagonal, window's end, sinks, padding) test their elements.  The backward recomputes S and dP in both passes
// (7 products for the 5 of a single pass), so no sum depends on the order of atomics.
//
// fp32 tensors are split exactly into three bf16 planes on the way into LDS and the products kept to fp32 level by six
// MFMAs (common.h, bf16x6).  bf16 tensors take one, and two where a factor is formed here: P and dS go into O, dV, dQ and
// dK as two bf16 terms (to 2^-16), whatever the sizes, so that an output is off by little beside its own rounding and a
// sequence's does not depend on what else is in its batch.  P in one term doubled the square of O's and dV's error (0.0023
// of the output in place of 0.0017; L = 8192 below: forward 246 us, dK and dV 500); dS in one, whose terms cancel (a row of
// it sums to 0), put dQ and dK off by 1.5 to 2 times their rounding.  Scores, softmax statistics and all sums are fp32.
// Measured: 2 sequences of 8192, 16 heads on 4, 128 columns, window 1024 and 4 sinks, causal, bf16: forward 279 us (460
// TFLOP/s of visible pairs, 40 % of what the library's large product reaches), dQ 369 (520), dK and dV 574 + 52 for what
// queries outside the window see of the sinks (410).  Counters (profiles/history_ops_counters.json), of forward, dQ and
// dK / dV: MFMA busy 29, 29 and 27 %, vector units 36, 29 and 25 %, LDS 13, 13 and 22 %, waves waiting 37, 45 and 52 % of
// their cycles; no bank conflicts.
#include "elem.h"

using namespace asme;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTS = 64;                  // streamed rows per tile
constexpr int kRowB = 256;               // bytes of a row of an LDS image
constexpr int kImage = kTS * kRowB;      // 16 KiB

typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4;

// byte of 16-byte chunk ch in row r of an image of 256-byte rows: transposed reads without bank conflicts, row reads 2-way
__device__ __forceinline__ int swz(int r, int ch) { return r * kRowB + 16 * (ch ^ (((r & 3) << 2) | ((r >> 2) & 3))); }

// NP planes of 8 values along k: an MFMA operand fragment
template <int NP>
struct Frag {
    bf16x8 p[NP];
};
__device__ __forceinline__ floatx16 product(const Frag<1>& a, const Frag<1>& b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 product(const Frag<3>& a, const Frag<3>& b, floatx16 c) {  // smallest terms first
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[2], b.p[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 product(const Frag<1>& a, const Frag<2>& b, floatx16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}
__device__ __forceinline__ Frag<2> frag_of(const float (&x)[8], Frag<2>*) {  // to 2^-16
    Frag<2> f;
    f.p[0] = Elem<__bf16>::pack(x);
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i] - (float)f.p[0][i];
    f.p[1] = Elem<__bf16>::pack(r);
    return f;
}
__device__ __forceinline__ Frag<1> frag_of(const float (&x)[8], Frag<1>*) { return {Elem<__bf16>::pack(x)}; }
__device__ __forceinline__ Frag<3> frag_of(const float (&x)[8], Frag<3>*) {
    const Bf3 s = split_bf3(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]));
    return {s.h, s.m, s.l};
}

// a tensor of (batch, token, head) rows of `dim` adjacent values
struct Tensor {
    void* p;
    int64_t sb, st, sh;
    template <class T>
    __device__ __forceinline__ T* at(int64_t b, int64_t h) const {
        return (T*)p + b * sb + h * sh;
    }
};

struct Args {
    Tensor q, k, v, out, dout, dq, dk, dv;
    const uint8_t* valid;  // (batch, seq_len) or null
    void* out_low;         // bf16 only, null or laid out like out: what rounding took from it
    float2* state;         // (batch, heads, seq_len): maximum of the scaled scores in base 2, 1 / sum
    float* delta;          // (batch, heads, seq_len): D
    float *part, *far_part;  // partial dK, dV: (key head, block, piece, 2, rows, dim), (key head, sinks, piece, 2, 64, dim)
    int seq_len, dim, heads, kv_heads, group, window, sinks, causal;
    int blocks;            // stationary blocks of a sequence
    uint32_t items, per_xcd;  // workgroups of the pass, those of an XCD
    // dK, dV: rows of a key block and its pieces; groups of 64 sinks that queries outside their block's tiles see (0: none
    // do), and the pieces of a group
    int near_rows, near_pieces, far_groups, far_pieces;
    float scale;
};

// values of 8 columns of a row, on their way to LDS
template <class T>
struct Chunk;
template <>
struct Chunk<float> {
    floatx4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const floatx4*>(p);
        b = *reinterpret_cast<const floatx4*>(p + 4);
    }
    __device__ __forceinline__ void zero() { a = b = floatx4{0.f, 0.f, 0.f, 0.f}; }
    __device__ __forceinline__ Frag<3> frag() const {
        const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        return frag_of(x, (Frag<3>*)nullptr);
    }
};
template <>
struct Chunk<__bf16> {
    bf16x8 a;
    __device__ __forceinline__ void load(const __bf16* p) { a = *reinterpret_cast<const bf16x8*>(p); }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = (__bf16)0.f;
    }
    __device__ __forceinline__ Frag<1> frag() const { return {a}; }
};

template <class T, int DP, int NW>
struct Pass {
    static constexpr int NP = sizeof(T) == 4 ? 3 : 1;
    static constexpr int KS = DP / 16, NFT = DP / 32;  // k steps of a score, 32-feature tiles of a gradient
    static constexpr int kThreads = NW * 64;
    static constexpr int kChunks = kTS * (DP / 8);      // 16-byte chunks of one tensor's tile (per plane)
    static constexpr int kEach = 2 * kChunks / kThreads;
    static constexpr int kRowStep = kThreads / (DP / 8);  // rows that the workgroup covers in one go
    static_assert(kChunks % kThreads == 0, "a thread's first chunks are of the first tensor, the others of the second");
    // two tensors side by side in one image up to 64 columns, in an image each at 128
    static constexpr int kImages = DP == 128 ? 2 : 1;
    static constexpr int kBytes = NP * kImages * kImage;
    using F = Frag<NP>;
    static constexpr int SP = NP == 1 ? 2 : NP;  // planes of P and dS as factors
    using S = Frag<SP>;

    // The compiler keeps the LDS addresses of a tile's reads and writes, which are the same in every round, in registers:
    // faster than forming them anew where there are registers (L = 8192, bf16, 128 columns: forward 378 us anew, 327 like
    // this, both by events; dK and dV the same, though 37 values of its eight-wave form spill like this).  fp32 rows of 128
    // columns leave none (up to 91 spilled values); there the thread's number is made new to it in every round.
    static __device__ __forceinline__ int thread() {
        int t = threadIdx.x;
        if constexpr (NP == 3 && DP == 128) asm volatile("" : "+v"(t));
        return t;
    }
    static __device__ __forceinline__ int place(int op, int plane, int row, int ch) {
        if constexpr (DP == 128) return (plane * 2 + op) * kImage + swz(row, ch);
        return plane * kImage + swz(row, ch + op * (DP / 8));
    }
    // is streamed position t0 + lane in the sequence and valid (the same in every wave)?  Read with the tile and looked
    // at when the tile is: a tile waits for one latency, not for two in a row
    static __device__ __forceinline__ int valid_row(const Args& a, int64_t b, int t0) {
        const int pos = t0 + (threadIdx.x & 63);
        if (pos >= a.seq_len) return 0;
        return a.valid ? a.valid[b * a.seq_len + pos] : 1;
    }
    // the tile's rows from t0 on of two tensors (base: their first row, uniform): a 32-bit offset per chunk, the same for
    // every whole tile.  Rows behind the sequence read its last one; put() clears them.
    static __device__ __forceinline__ void fetch(Chunk<T> (&c)[kEach], const T* x0, int64_t st0, const T* x1,
                                                 int64_t st1, int t0, int seq_len, int dim) {
        const T *b0 = x0 + t0 * st0, *b1 = x1 + t0 * st1;
        const int ch = threadIdx.x % (DP / 8) * 8;
        const bool in = DP > 32 || ch < dim;  // (a head of 16 leaves the second half of 32 columns empty)
        if (t0 + kTS <= seq_len) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const uint32_t row = e % (kEach / 2) * kRowStep + threadIdx.x / (DP / 8);
                c[e].zero();
                if (in) c[e].load(e < kEach / 2 ? b0 + (row * (uint32_t)st0 + ch) : b1 + (row * (uint32_t)st1 + ch));
            }
        } else {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const uint32_t row = min(e % (kEach / 2) * kRowStep + (int)threadIdx.x / (DP / 8), seq_len - 1 - t0);
                c[e].zero();
                if (in) c[e].load(e < kEach / 2 ? b0 + (row * (uint32_t)st0 + ch) : b1 + (row * (uint32_t)st1 + ch));
            }
        }
    }
    static __device__ __forceinline__ void put(char* lds, Chunk<T> (&c)[kEach], uint64_t rows) {
        const int t = thread(), ch = t % (DP / 8);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int row = e % (kEach / 2) * kRowStep + t / (DP / 8);
            if (rows != ~0ull && !((rows >> row) & 1)) c[e].zero();
            const F f = c[e].frag();
#pragma unroll
            for (int p = 0; p < NP; ++p)
                *reinterpret_cast<bf16x8*>(lds + place(e < kEach / 2 ? 0 : 1, p, row, ch)) = f.p[p];
        }
    }
    // stationary fragments of row `row` (null: zeros)
    static __device__ __forceinline__ void stationary(F (&f)[KS], const T* row, int h, int dim) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            Chunk<T> c;
            if (row && 16 * ks + 8 * h < dim) c.load(row + 16 * ks + 8 * h);
            else c.zero();
            f[ks] = c.frag();
        }
    }
    // X[streamed row of the 32-row half `sub`][stationary row] of tensor `op`.  The reads of kStep k steps are issued
    // together, so that a product waits for the first of them and not each for its own
    static constexpr int kStep = NP == 1 ? (KS < 4 ? KS : 4) : 2;
    static __device__ __forceinline__ floatx16 score(const char* lds, int op, int sub, const F (&st)[KS]) {
        const int lane = thread() & 63, r32 = lane & 31, h = lane >> 5;
        floatx16 x;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.f;
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += kStep) {
            F A[kStep];
#pragma unroll
            for (int ks = 0; ks < kStep; ++ks)
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    A[ks].p[p] = *reinterpret_cast<const bf16x8*>(lds + place(op, p, 32 * sub + r32, 2 * (k0 + ks) + h));
#pragma unroll
            for (int ks = 0; ks < kStep; ++ks) x = product(A[ks], st[k0 + ks], x);
        }
        return x;
    }
    // Y^T[feature][stationary row] += streamed^T . x: rows 16 s2 + 8 (j >> 2) + 4 h + (j & 3) of the half are element j of
    // the lane's B fragment; 16-lane group (h, fh) reads rows + q x features 32 ft + 16 fh + 4 p4 .. + 3 transposed
    template <int N>
    static __device__ __forceinline__ void read_transposed(const char* lds, int op, int sub, int s2, int first, F (&A)[N]) {
        const int lane = thread() & 63, h = lane >> 5, fh = (lane >> 4) & 1, q = (lane & 15) >> 2, p4 = lane & 3;
        const int lo = 32 * sub + 16 * s2 + 4 * h + q;
#pragma unroll
        for (int ft = 0; ft < N; ++ft) {
            const int ch = 4 * (first + ft) + 2 * fh + (p4 >> 1);
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_short4*)(lds + place(op, p, lo, ch) + 8 * (p4 & 1)));
                const short4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_short4*)(lds + place(op, p, lo + 8, ch) + 8 * (p4 & 1)));
                typedef short short8v __attribute__((ext_vector_type(8)));
                const short8v c = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                A[ft].p[p] = __builtin_bit_cast(bf16x8, c);
            }
        }
    }
    template <class W>
    static __device__ __forceinline__ W weights_of(const floatx16& x, int s2) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x[8 * s2 + j];
        return frag_of(v, (W*)nullptr);
    }
    // Y^T[features from 32 `first` on] += streamed^T . w of k step s2
    template <class W, int N>
    static __device__ __forceinline__ void gather(const char* lds, int op, int sub, int s2, int first, const W& w,
                                                  floatx16 (&y)[N]) {
        F A[N];
        read_transposed(lds, op, sub, s2, first, A);
#pragma unroll
        for (int ft = 0; ft < N; ++ft) y[ft] = product(A[ft], w, y[ft]);
    }
    // a fragment in lane order: plane p is 1 KiB at `at` + p KiB
    template <int N>
    static __device__ __forceinline__ void pass_on(char* at, const Frag<N>& w) {
#pragma unroll
        for (int p = 0; p < N; ++p) *reinterpret_cast<bf16x8*>(at + p * 1024) = w.p[p];
    }
    template <class W>
    static __device__ __forceinline__ W passed(const char* at) {
        W w;
#pragma unroll
        for (int p = 0; p < (int)(sizeof(W) / sizeof(bf16x8)); ++p)
            w.p[p] = *reinterpret_cast<const bf16x8*>(at + p * 1024);
        return w;
    }
    // row `row` (features 32 ft + 8 i + 4 h .. + 3 of this lane's stationary row) = y * f
    template <int N>
    static __device__ __forceinline__ void write_row(T* row, const floatx16 (&y)[N], float f, int h, int dim) {
#pragma unroll
        for (int ft = 0; ft < N; ++ft)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 32 * ft + 8 * i + 4 * h;
                if (c >= dim) continue;
                if constexpr (NP == 3) {
                    *reinterpret_cast<floatx4*>(row + c) = floatx4{y[ft][4 * i] * f, y[ft][4 * i + 1] * f,
                                                                   y[ft][4 * i + 2] * f, y[ft][4 * i + 3] * f};
                } else {
                    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                    *reinterpret_cast<bf16x4*>(row + c) =
                        bf16x4{(__bf16)(y[ft][4 * i] * f), (__bf16)(y[ft][4 * i + 1] * f),
                               (__bf16)(y[ft][4 * i + 2] * f), (__bf16)(y[ft][4 * i + 3] * f)};
                }
            }
    }
    // low = what rounding takes from y * f where write_row() stores it
    template <int N>
    static __device__ __forceinline__ void write_low(__bf16* row, const floatx16 (&y)[N], float f, int h, int dim) {
#pragma unroll
        for (int ft = 0; ft < N; ++ft)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 32 * ft + 8 * i + 4 * h;
                if (c >= dim) continue;
                typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                bf16x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = y[ft][4 * i + e] * f;
                    v[e] = (__bf16)(x - (float)(__bf16)x);
                }
                *reinterpret_cast<bf16x4*>(row + c) = v;
            }
    }
    // y += f * a row of fp32 values laid out like that
    template <int N>
    static __device__ __forceinline__ void add_row(const float* row, floatx16 (&y)[N], float f, int h, int dim) {
        floatx4 x[N][4];
#pragma unroll
        for (int ft = 0; ft < N; ++ft)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 32 * ft + 8 * i + 4 * h;
                x[ft][i] = *reinterpret_cast<const floatx4*>(row + (DP > 32 || c < dim ? c : 0));
            }
#pragma unroll
        for (int ft = 0; ft < N; ++ft)
#pragma unroll
            for (int e = 0; e < 16; ++e) y[ft][e] = fmaf(f, x[ft][e >> 2][e & 3], y[ft][e]);
    }
    template <int N>
    static __device__ __forceinline__ void clear(floatx16 (&y)[N]) {
#pragma unroll
        for (int f = 0; f < N; ++f)
#pragma unroll
            for (int i = 0; i < 16; ++i) y[f][i] = 0.f;
    }
};

// bits 0 .. n (none for n < 0, all from n = 31 on)
__device__ __forceinline__ uint32_t upto(int n) { return n < 0 ? 0u : n >= 31 ? ~0u : (2u << n) - 1u; }
// bit r: query i sees key j0 + r
__device__ __forceinline__ uint32_t keys_seen(const Args& a, int i, int j0) {
    const uint32_t after = ~upto(i - a.window - j0), sinks = upto(a.sinks - 1 - j0);  // j > i - window; j < sinks
    if (a.causal) return upto(i - j0) & (after | sinks);
    return (upto(i + a.window - 1 - j0) & after) | sinks;
}
// bit r: query i0 + r sees key j
__device__ __forceinline__ uint32_t queries_seen(const Args& a, int i0, int j) {
    const uint32_t before = j < a.sinks ? ~0u : upto(j + a.window - 1 - i0);  // i < j + window, or any
    if (a.causal) return before & ~upto(j - 1 - i0);
    return j < a.sinks ? ~0u : before & ~upto(j - a.window - i0);
}
// bit of accumulator register e among the 32 rows' bits, those shifted down by 4 h
__device__ __forceinline__ bool row_bit(uint32_t bits, int e) { return (bits >> ((e & 3) + 8 * (e >> 2))) & 1u; }
// The block of queries i0 .. i0 + 31 and keys j0 .. j0 + 31, by its corners: 0 no pair visible, 2 every pair, 1 some
__device__ __forceinline__ int block_seen(const Args& a, int i0, int j0) {
    const int most = i0 + 31 - j0, least = i0 - (j0 + 31);  // i - j over the block
    if (a.causal) {
        if (most < 0) return 0;
        if (least >= 0 && (most < a.window || j0 + 31 < a.sinks)) return 2;
        return least >= a.window && j0 >= a.sinks ? 0 : 1;
    }
    if ((most < a.window && -least < a.window) || j0 + 31 < a.sinks) return 2;
    return (least >= a.window || -most >= a.window) && j0 >= a.sinks ? 0 : 1;
}

// workgroup -> item: neighbours (blocks of the same head, which read the same streamed rows) on one XCD, so that they
// share its L2 (the dispatcher deals workgroups round-robin over the 8 XCDs; only a matter of speed)
__device__ __forceinline__ bool item_of(const Args& a, uint32_t& item) {
    item = blockIdx.x % 8 * a.per_xcd + blockIdx.x / 8;
    return item < a.items;
}

// The streamed key tiles of queries [q0, q1): those of the sinks in front of the window's first tile, then the window's,
// without causal up to the last sink where that lies beyond the window (every key in between is a sink).
struct KeyTiles {
    int sink_tiles, lo, count;
    __device__ KeyTiles(const Args& a, int q0, int q1) {
        lo = max(0, q0 - a.window + 1) / kTS * kTS;
        const int hi = a.causal ? q1 : max(a.sinks, (int)min((int64_t)a.seq_len, (int64_t)q1 - 1 + a.window));
        sink_tiles = (min(a.sinks, lo) + kTS - 1) / kTS;
        count = sink_tiles + (hi - lo + kTS - 1) / kTS;
    }
    __device__ int start(int i) const { return i < sink_tiles ? i * kTS : lo + (i - sink_tiles) * kTS; }
};

// ------------------------------------------------------------------------------------------------ forward
template <class T, int DP, int NW>
__global__ __launch_bounds__(NW * 64) void forward_kernel(Args a) {
    using P = Pass<T, DP, NW>;
    __shared__ __attribute__((aligned(16))) char lds[P::kBytes];
    uint32_t item;
    if (!item_of(a, item)) return;  // (the whole workgroup)
    const int lane = threadIdx.x & 63, h = lane >> 5, r32 = lane & 31;
    const uint32_t row = item / (uint32_t)a.blocks;  // sequence and head
    const int block = (int)(item - row * a.blocks), head = (int)(row % (uint32_t)a.heads);
    const int64_t b = row / (uint32_t)a.heads;
    const int q0 = block * NW * 32, q1 = min(a.seq_len, q0 + NW * 32);
    const int w0 = q0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 32, qi = w0 + r32;
    const bool live = qi < a.seq_len && (!a.valid || a.valid[b * a.seq_len + qi]);
    const bool any = __ballot(live) != 0;
    typename P::F Q[P::KS];
    P::stationary(Q, live ? a.q.at<T>(b, head) + qi * a.q.st : nullptr, h, a.dim);
    floatx16 y[P::NFT];
    P::clear(y);
    float top = -INFINITY, sum = 0.f;
    const float c = a.scale * kLog2e;
    const T* K = a.k.at<T>(b, head / a.group);
    const T* V = a.v.at<T>(b, head / a.group);
    const KeyTiles tiles(a, q0, q1);
    Chunk<T> next[P::kEach];
    int i = 0, t0 = 0, valid = 0;
    auto issue = [&]() {  // tile i, on its way
        if (i >= tiles.count) return;
        t0 = tiles.start(i);
        valid = P::valid_row(a, b, t0);
        P::fetch(next, K, a.k.st, V, a.v.st, t0, a.seq_len, a.dim);
    };
    if (__syncthreads_or(any)) issue();
    else i = tiles.count;
    while (i < tiles.count) {
        const int k0 = t0;
        const uint64_t keys = __ballot(valid != 0);
        __syncthreads();  // the last tile has been read
        P::put(lds, next, keys);
        __syncthreads();
        ++i;
        issue();
        if (!any) continue;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const uint32_t ok = (uint32_t)(keys >> (32 * sub));
            const int j0 = k0 + 32 * sub, seen = ok ? block_seen(a, w0, j0) : 0;
            if (!seen) continue;
            floatx16 x = P::score(lds, 0, sub, Q);
            if (seen == 1 || ok != 0xFFFFFFFFu) {
                const uint32_t bits = (ok & keys_seen(a, qi, j0)) >> (4 * h);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = row_bit(bits, e) ? x[e] : -INFINITY;
            }
            float t = x[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) t = fmaxf(t, x[e]);
            t = fmaxf(t, __shfl_xor(t, 32, 64)) * c;
            // the reference moves only when some row's maximum passes it by more than 8: P <= 2^8 in between
            if (__ballot(!(t <= top + 8.f)) != 0ull) {
                const float m = fmaxf(top, t), f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - m);
#pragma unroll
                for (int ft = 0; ft < P::NFT; ++ft)
#pragma unroll
                    for (int e = 0; e < 16; ++e) y[ft][e] *= f;
                sum *= f;
                top = m;
            }
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], c, -base));
                sum += x[e];
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
                P::gather(lds, 1, sub, s2, 0, P::template weights_of<typename P::S>(x, s2), y);
        }
    }
    sum += __shfl_xor(sum, 32, 64);
    if (qi >= a.seq_len) return;
    const float inv = live ? 1.f / sum : 0.f;
    if (!live) P::clear(y);
    P::write_row(a.out.at<T>(b, head) + qi * a.out.st, y, inv, h, a.dim);
    if constexpr (sizeof(T) == 2)
        if (a.out_low) P::write_low((T*)a.out_low + b * a.out.sb + head * a.out.sh + qi * a.out.st, y, inv, h, a.dim);
    // a position that is no query: P = 2^-inf = 0 in the backward
    if (a.state && h == 0) a.state[(b * a.heads + head) * a.seq_len + qi] = make_float2(live ? top : INFINITY, inv);
}

// ------------------------------------------------------------------------------------------------ dQ
template <class T, int DP, int NW>
__global__ __launch_bounds__(NW * 64) void dq_kernel(Args a) {
    using P = Pass<T, DP, NW>;
    __shared__ __attribute__((aligned(16))) char lds[P::kBytes];
    uint32_t item;
    if (!item_of(a, item)) return;
    const int lane = threadIdx.x & 63, h = lane >> 5, r32 = lane & 31;
    const uint32_t row = item / (uint32_t)a.blocks;  // sequence and head
    const int block = (int)(item - row * a.blocks), head = (int)(row % (uint32_t)a.heads);
    const int64_t b = row / (uint32_t)a.heads;
    const int q0 = block * NW * 32, q1 = min(a.seq_len, q0 + NW * 32);
    const int w0 = q0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 32, qi = w0 + r32;
    const bool live = qi < a.seq_len && (!a.valid || a.valid[b * a.seq_len + qi]);
    const bool any = __ballot(live) != 0;
    typename P::F Q[P::KS], O[P::KS];
    P::stationary(Q, live ? a.q.at<T>(b, head) + qi * a.q.st : nullptr, h, a.dim);
    P::stationary(O, live ? a.dout.at<T>(b, head) + qi * a.dout.st : nullptr, h, a.dim);
    // D of the row: each half of the lanes holds half of its columns.  O with what its rounding took: D is the same number
    // for every key of the row, so that its error would not average out of dQ and dK as the rounding of dS does
    float delta = 0.f;
    if (live) {
        const T* o = a.out.at<T>(b, head) + qi * a.out.st;
        const T* d = a.dout.at<T>(b, head) + qi * a.dout.st;
        const T* low = a.out_low ? (const T*)a.out_low + (o - (const T*)a.out.p) : nullptr;
#pragma unroll
        for (int ks = 0; ks < P::KS; ++ks) {
            if (16 * ks >= a.dim) continue;
            constexpr int E = Elem<T>::V;
#pragma unroll
            for (int e = 0; e < 8; e += E) {
                float x[E], z[E];
                Elem<T>::load(o + 16 * ks + 8 * h + e, x);
                Elem<T>::load(d + 16 * ks + 8 * h + e, z);
#pragma unroll
                for (int k = 0; k < E; ++k) delta = fmaf(x[k], z[k], delta);
                if (low) {
                    Elem<T>::load(low + 16 * ks + 8 * h + e, x);
#pragma unroll
                    for (int k = 0; k < E; ++k) delta = fmaf(x[k], z[k], delta);
                }
            }
        }
    }
    delta += __shfl_xor(delta, 32, 64);
    const int64_t at = (b * a.heads + head) * a.seq_len + qi;
    float2 st = make_float2(INFINITY, 0.f);
    if (live) st = a.state[at];
    if (qi < a.seq_len && h == 0) a.delta[at] = delta;
    floatx16 y[P::NFT];
    P::clear(y);
    const float c = a.scale * kLog2e;
    const T* K = a.k.at<T>(b, head / a.group);
    const T* V = a.v.at<T>(b, head / a.group);
    const KeyTiles tiles(a, q0, q1);
    Chunk<T> next[P::kEach];
    int i = 0, t0 = 0, valid = 0;
    auto issue = [&]() {  // tile i, on its way
        if (i >= tiles.count) return;
        t0 = tiles.start(i);
        valid = P::valid_row(a, b, t0);
        P::fetch(next, K, a.k.st, V, a.v.st, t0, a.seq_len, a.dim);
    };
    if (__syncthreads_or(any)) issue();
    else i = tiles.count;
    while (i < tiles.count) {
        const int k0 = t0;
        const uint64_t keys = __ballot(valid != 0);
        __syncthreads();  // the last tile has been read
        P::put(lds, next, keys);
        __syncthreads();
        ++i;
        issue();
        if (!any) continue;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const uint32_t ok = (uint32_t)(keys >> (32 * sub));
            const int j0 = k0 + 32 * sub, seen = ok ? block_seen(a, w0, j0) : 0;
            if (!seen) continue;
            floatx16 x = P::score(lds, 0, sub, Q);
            const floatx16 dp = P::score(lds, 1, sub, O);
            if (seen == 1 || ok != 0xFFFFFFFFu) {
                const uint32_t bits = (ok & keys_seen(a, qi, j0)) >> (4 * h);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = row_bit(bits, e) ? x[e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e)
                x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], c, -st.x)) * st.y * (dp[e] - delta);
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
                P::gather(lds, 0, sub, s2, 0, P::template weights_of<typename P::S>(x, s2), y);
        }
    }
    if (qi >= a.seq_len) return;
    if (!live) P::clear(y);
    P::write_row(a.dq.at<T>(b, head) + qi * a.dq.st, y, a.scale, h, a.dim);
}

// ------------------------------------------------------------------------------------------------ dK, dV
// The query tiles that the near pass of the key block from k0 on streams: those that a key of the block is in the window
// of.  What a sink is seen by beyond them is the far pass's.
struct QueryTiles {
    int lo, hi;
    // without a far pass, a block with sinks takes all
    __host__ __device__ QueryTiles(const Args& a, int k0, int rows) {
        if (a.far_groups == 0 && k0 < a.sinks) {
            lo = a.causal ? k0 / kTS : 0, hi = (a.seq_len + kTS - 1) / kTS;
            return;
        }
        const int64_t k1 = k0 + rows < a.seq_len ? k0 + rows : a.seq_len, end = k1 - 1 + a.window;
        const int first = a.causal ? k0 : k0 - a.window + 1;
        lo = first > 0 ? first / kTS : 0;
        hi = (int)(((end < a.seq_len ? end : a.seq_len) + kTS - 1) / kTS);
    }
};

// Two waves hold the same 32 keys.  Each forms P and dS of its half of the tile's queries and passes them on; each sums dK
// and dV over all the queries, for its half of the columns.  With all columns in one wave the pass needs over 256 registers
// at 128 columns and runs at one wave per SIMD, where the matrix and vector units take turns; with all of dV in one wave and
// all of dK in the other, dS's second term would be a branch (800 us for L = 8192 in bf16, P in one term; 500 like this).  Heads
// of 32 columns have no halves: there a wave sums its half of the queries, and the pair adds up at the end.
constexpr int kFarWaves = 4, kFarRows = 16 * kFarWaves;  // sinks of a workgroup of the far pass
// where the far pass's sums of dK (0) or dV (1) of key kj begin
__device__ __forceinline__ int64_t far_row(const Args& a, int64_t bk, int kj, int which) {
    return ((bk * a.far_groups + kj / kFarRows) * a.far_pieces * 2 * kFarRows + which * kFarRows + kj % kFarRows) * a.dim;
}

// Near item: (sequence, key head, block of NW x 16 keys, piece); its steps are the block's query tiles for each query head
// of the group, of which a piece takes a contiguous share.  One piece: dK and dV at once, the far pass's rows added; else
// partial rows.
// Far item: (sequence, key head, NW x 16 sinks, piece) over the query tiles outside the near pass's of the sinks' block,
// into partial rows.
template <class T, int DP, int NW, bool FAR>
__global__ __launch_bounds__(NW * 64) void dkv_kernel(Args a) {
    using P = Pass<T, DP, NW>;
    using S = typename P::S;
    constexpr bool kHalves = DP > 32;
    constexpr int N = kHalves ? P::NFT / 2 : 1;
    constexpr int kS = 64 * sizeof(S);  // bytes of a wave's P or dS of a k step
    constexpr int kPassed = kHalves ? 4 * kS : 64 * sizeof(floatx16);
    __shared__ __attribute__((aligned(16))) char lds[P::kBytes];
    __shared__ __attribute__((aligned(16))) char exchange[NW * kPassed];  // P, dS of a wave's half; or a sum
    __shared__ __attribute__((aligned(16))) float meta[3][kTS];  // maximum, 1 / sum, D of the tile's queries
    uint32_t item;
    if (!item_of(a, item)) return;
    const int lane = threadIdx.x & 63, h = lane >> 5, r32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), role = wave & 1;
    const int pieces = FAR ? a.far_pieces : a.near_pieces;
    const uint32_t unit = item / (uint32_t)pieces, per_head = FAR ? a.far_groups : a.blocks, bk = unit / per_head;
    const int piece = (int)(item - unit * pieces), block = (int)(unit - bk * per_head);
    const int kh = (int)(bk % (uint32_t)a.kv_heads);
    const int64_t b = bk / (uint32_t)a.kv_heads;
    const int w0 = block * NW * 16 + (wave >> 1) * 32, kj = w0 + r32;
    const bool live = kj < a.seq_len && (!FAR || kj < a.sinks) && (!a.valid || a.valid[b * a.seq_len + kj]);
    const bool any = __ballot(live) != 0;
    const uint32_t ok = (uint32_t)__ballot(live);  // (both halves of the lanes hold the same keys)
    typename P::F K[P::KS], V[P::KS];
    P::stationary(K, live ? a.k.at<T>(b, kh) + kj * a.k.st : nullptr, h, a.dim);
    P::stationary(V, live ? a.v.at<T>(b, kh) + kj * a.v.st : nullptr, h, a.dim);
    floatx16 yv[N], yk[N];
    P::clear(yv), P::clear(yk);
    const int first = kHalves ? role * N : 0;
    const float c = a.scale * kLog2e;
    const QueryTiles near(a, block * NW * 16 / a.near_rows * a.near_rows, a.near_rows);
    // the near tiles, or those beside them: [0, lo) without causal, and [hi, all)
    const int before = FAR && !a.causal ? near.lo : 0, jump = FAR ? near.hi : near.lo;
    const int tiles = FAR ? before + (a.seq_len + kTS - 1) / kTS - near.hi : near.hi - near.lo, steps = tiles * a.group;
    int i = (int)((int64_t)steps * piece / pieces), t0 = 0;
    const int last = (int)((int64_t)steps * (piece + 1) / pieces);
    int valid = 0;
    Chunk<T> next[P::kEach];
    float2 st = make_float2(INFINITY, 0.f);
    float delta = 0.f;
    auto issue = [&]() {
        if (i >= last) return;
        const int tile = i % tiles, head = kh * a.group + i / tiles;
        t0 = (tile < before ? tile : tile - before + jump) * kTS;
        valid = P::valid_row(a, b, t0);
        P::fetch(next, a.q.at<T>(b, head), a.q.st, a.dout.at<T>(b, head), a.dout.st, t0, a.seq_len, a.dim);
        if (threadIdx.x < kTS) {  // (of a query that is none: (infinity, 0) and 0)
            const int64_t at = (b * a.heads + head) * a.seq_len + t0 + threadIdx.x;
            st = make_float2(INFINITY, 0.f), delta = 0.f;
            if (t0 + (int)threadIdx.x < a.seq_len) st = a.state[at], delta = a.delta[at];
        }
    };
    char* mine = exchange + wave * kPassed + lane * 16;
    const char* other = exchange + (wave ^ 1) * kPassed + lane * 16;
    if (__syncthreads_or(any)) issue();
    else i = last;
    while (i < last) {
        const int q0 = t0;
        const uint64_t queries = __ballot(valid != 0);
        __syncthreads();
        P::put(lds, next, queries);
        if (threadIdx.x < kTS) meta[0][threadIdx.x] = st.x, meta[1][threadIdx.x] = st.y, meta[2][threadIdx.x] = delta;
        __syncthreads();
        ++i;
        issue();
        auto seen_of = [&](int sub) {
            return any && (uint32_t)(queries >> (32 * sub)) ? block_seen(a, q0 + 32 * sub, w0) : 0;
        };
        const int seen = seen_of(role), theirs = kHalves ? seen_of(role ^ 1) : 0;
        if (seen) {
            floatx16 x = P::score(lds, 0, role, K);
            floatx16 dp = P::score(lds, 1, role, V);
            if (seen == 1 || ok != 0xFFFFFFFFu) {
                const uint32_t bits = live ? queries_seen(a, q0 + 32 * role, kj) >> (4 * h) : 0u;
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = row_bit(bits, e) ? x[e] : -INFINITY;
            }
            const float* m = &meta[0][32 * role + 4 * h];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int r = 8 * (e >> 2) + (e & 3);
                x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], c, -m[r])) * m[kTS + r];
                dp[e] = x[e] * (dp[e] - m[2 * kTS + r]);
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                const auto w = P::template weights_of<S>(x, s2);
                if constexpr (kHalves) P::pass_on(mine + s2 * kS, w);
                P::gather(lds, 1, role, s2, first, w, yv);
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                const auto w = P::template weights_of<S>(dp, s2);
                if constexpr (kHalves) P::pass_on(mine + (2 + s2) * kS, w);
                P::gather(lds, 0, role, s2, first, w, yk);
            }
        }
        if constexpr (!kHalves) continue;
        __syncthreads();
        if (theirs) {
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
                P::gather(lds, 1, role ^ 1, s2, first, P::template passed<S>(other + s2 * kS), yv);
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
                P::gather(lds, 0, role ^ 1, s2, first, P::template passed<S>(other + (2 + s2) * kS), yk);
        }
    }
    if constexpr (!kHalves) {  // the first wave takes dV, the second dK
        floatx16 *give = (floatx16*)exchange + wave * 64 + lane, *take = (floatx16*)exchange + (wave ^ 1) * 64 + lane;
        __syncthreads();
        *give = role ? yv[0] : yk[0];
        __syncthreads();
        yv[0] = (role ? yk[0] : yv[0]) + *take;
    }
    using PF = Pass<float, DP, NW>;
    // f(dK?, the sum, its first column): what of the two rows this wave holds
    auto each = [&](auto f) {
        if (kHalves || !role) f(0, yv, 32 * first);
        if (kHalves) f(1, yk, 32 * first);
        else if (role) f(1, yv, 0);
    };
    if (FAR || pieces > 1) {  // slab (key head, block, piece): dK and dV of the block's rows, zeros where there is nothing
        each([&](int is_k, auto& y, int col) {
            PF::write_row((FAR ? a.far_part : a.part) +
                              (((int64_t)item * 2 + !is_k) * NW * 16 + (wave >> 1) * 32 + r32) * a.dim + col,
                          y, is_k ? a.scale : 1.f, h, a.dim - col);
        });
        return;
    }
    if (kj >= a.seq_len) return;
    each([&](int is_k, auto& y, int col) {
        const float f = is_k ? a.scale : 1.f;
        if (w0 < kFarRows * a.far_groups)  // the far pass's sums, added up in its first slab (0 for rows that are no sinks)
            P::add_row(a.far_part + far_row(a, bk, kj, !is_k) + col, y, 1.f / f, h, a.dim - col);
        if (!live) P::clear(y);
        const Tensor& t = is_k ? a.dk : a.dv;
        P::write_row(t.at<T>(b, kh) + kj * t.st + col, y, f, h, a.dim - col);
    });
}

// the far pass's slabs of a group of sinks added up in the first, in order, 4 columns a thread
__global__ __launch_bounds__(256) void add_far_kernel(float* part, int slabs, int dim, int64_t total) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t slab = 2 * kFarRows * dim, quads = slab / 4;
    float* p = part + i / quads * slabs * slab + i % quads * 4;
    floatx4 s = *reinterpret_cast<const floatx4*>(p);
#pragma unroll 8
    for (int u = 1; u < slabs; ++u) s += *reinterpret_cast<const floatx4*>(p + u * slab);
    *reinterpret_cast<floatx4*>(p) = s;
}

// dK, dV of blocks in pieces: the near pass's partial rows and the far pass's added in order, 4 columns a thread
template <class T>
__global__ __launch_bounds__(256) void add_pieces_kernel(Args a, int64_t total) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int quads = a.dim / 4, c = (int)(i % quads) * 4, kj = (int)(i / quads % a.seq_len);
    const int64_t u = i / quads / a.seq_len, bk = u / 2, b = bk / a.kv_heads;
    const int which = (int)(u % 2), kh = (int)(bk % a.kv_heads), block = kj / a.near_rows, row = kj % a.near_rows;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](const float* p) {
        float x[4];
        Elem<float>::load(p, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += x[e];
    };
    if (!a.valid || a.valid[b * a.seq_len + kj]) {
        for (int p = 0; p < a.near_pieces; ++p)
            add(a.part + ((((bk * a.blocks + block) * a.near_pieces + p) * 2 + which) * a.near_rows + row) * a.dim + c);
        if (kj < kFarRows * a.far_groups)
            add(a.far_part + far_row(a, bk, kj, which) + c);
    }
    const Tensor& t = which ? a.dv : a.dk;
    T* o = t.at<T>(b, kh) + kj * t.st + c;
#pragma unroll
    for (int e = 0; e < 4; ++e) Elem<T>::put(o + e, s[e]);
}

// ------------------------------------------------------------------------------------------------ host
int padded_dim(int64_t dim) { return dim <= 32 ? 32 : (int)dim; }

// Waves (of 32 stationary rows) per workgroup: eight share a streamed tile's way through LDS, at 256 registers each; four
// (512 registers) where a pass's fragments and sums need more; two where the sequence has no more rows; half of them, twice
// if need be, where each workgroup still has a CU of its own (one sequence of 2000, 4 heads of 128 columns, window 256,
// bf16: forward 32 us, dQ 37 in 32 workgroups of eight waves, 21 and 22 in 126 of two; beyond that the tiles' way costs
// more: 3 of 2049, 6 heads of 64, fp32, 63 us in 162 of eight, 70 in 306 of four).
int waves(int64_t seqs, int64_t seq_len, int dtype, int dp) {  // seqs: sequences and heads
    int w = seq_len <= 64 ? 2 : dp == 32 || (dtype == kF32 && dp == 128) ? 4 : 8;
    while (w > 2 && seqs * ((seq_len + 16 * w - 1) / (16 * w)) <= 256) w /= 2;
    return w;
}
int waves_kv(int64_t seq_len, int dtype, int dp) {  // (two to 32 rows)
    return seq_len <= 64 || dp == 32 || (dtype == kF32 && dp == 128) ? 4 : 8;
}

// Pieces of the dK, dV passes.  Near: those that end first when the card takes its workgroups in rounds of `slots` and one
// costs its steps and about 3 more (its keys, its sums; 4 with the rows it leaves to be added); at least 4 steps each, at
// most 8 rounds (the partial rows' memory).  290 blocks in one piece are two rounds, the second nearly empty: 29 sequences
// of 1181, window 307 to both sides, four heads of 128 columns on one in bf16 take 345 us, in pieces 275 and 20 to add them
// up.  Far: as many as give every CU two
// workgroups, of at least 4 tiles; none where kAlong tiles or fewer are left to it, which the near pass takes along (256
// ragged sequences of up to 200, 2 heads of 64, window 64, fp32: 114 us with a far pass, 92 without).
constexpr int kAlong = 4;
void plan_kv(Args& a, int64_t batch, int dtype) {
    const int dp = padded_dim(a.dim), nw = waves_kv(a.seq_len, dtype, dp);
    const int64_t slots = 256 * (nw == 8 || (dtype == kF32 && dp > 32) ? 1 : 2);  // (by the waves that registers allow)
    a.near_rows = nw * 16;
    a.blocks = (a.seq_len + a.near_rows - 1) / a.near_rows;
    const int64_t have = batch * a.kv_heads, all = (a.seq_len + kTS - 1) / kTS;
    const int64_t reach = std::min<int64_t>(a.seq_len, a.near_rows + (int64_t)a.window * (a.causal ? 1 : 2));
    a.far_groups = (a.sinks + kFarRows - 1) / kFarRows;
    int64_t most = 0;  // tiles beside the near pass's, of the block that has the most
    for (int k0 = 0; k0 < a.sinks; k0 += a.near_rows) {
        const QueryTiles t(a, k0, a.near_rows);
        most = std::max<int64_t>(most, all - t.hi + (a.causal ? 0 : t.lo));
    }
    if (most * a.group <= kAlong) a.far_groups = 0;
    const int64_t steps = (reach + kTS - 1) / kTS * a.group;
    a.near_pieces = 1;
    int64_t best = INT64_MAX;
    for (int p = 1; p == 1 || (p <= 64 && steps / p >= 4 && have * a.blocks * p <= 8 * slots); ++p) {
        const int64_t rounds = (have * a.blocks * p + slots - 1) / slots, cost = rounds * ((steps + p - 1) / p + 3 + (p > 1));
        if (cost < best) best = cost, a.near_pieces = p;
    }
    a.far_pieces = a.far_groups ? (int)std::max<int64_t>(
        1, std::min<int64_t>({512 / (have * a.far_groups), most * a.group / 4, 64})) : 1;
}
int64_t slab_floats(const Args& a, int64_t batch) {
    return a.near_pieces > 1 ? batch * a.kv_heads * a.blocks * a.near_pieces * 2 * a.near_rows * a.dim : 0;
}
int64_t far_floats(const Args& a, int64_t batch) {
    return batch * a.kv_heads * a.far_groups * a.far_pieces * 2 * kFarRows * a.dim;
}

bool sizes_ok(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_len, int64_t dim, int64_t window,
              int64_t sinks) {
    return batch >= 1 && kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && seq_len >= 1 &&
           seq_len <= (1 << 24) && (dim == 16 || dim == 32 || dim == 64 || dim == 128) && window >= 1 && sinks >= 0 &&
           heads <= 65536 && batch <= (1ll << 24) && batch * heads * seq_len <= (1ll << 34);
}

bool strides_ok(const Tensor& t, int64_t per) {
    return t.p && ((uintptr_t)t.p & 15) == 0 && t.sb % per == 0 && t.st % per == 0 && t.sh % per == 0 && t.st >= 0 &&
           t.st < (1 << 23);  // (a tile's 64 rows are addressed by 32-bit offsets)
}

Args make_args(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_len, int64_t dim, int64_t window,
               int64_t sinks, int causal, float scale, const uint8_t* valid) {
    Args a{};
    a.seq_len = (int)seq_len, a.dim = (int)dim, a.heads = (int)heads, a.kv_heads = (int)kv_heads;
    a.group = (int)(heads / kv_heads), a.causal = causal, a.scale = scale, a.valid = valid;
    // a window or sinks longer than the sequence see all of it: 32-bit positions from here on
    a.window = (int)std::min(window, seq_len), a.sinks = (int)std::min(sinks, seq_len);
    return a;
}

Tensor tensor(const void* p, const int64_t* s) { return Tensor{const_cast<void*>(p), s[0], s[1], s[2]}; }

// f(T{}, DP, NW as integral constants)
template <class F>
void with_pass(int dtype, int dp, int nw, F&& f) {
    with_dtype(dtype, [&](auto t) {
        auto dim = [&](auto d) {
            // (the workgroup sizes that waves() and waves_kv() give)
            constexpr int most = decltype(d)::value == 32 || (sizeof(t) == 4 && decltype(d)::value == 128) ? 4 : 8;
            if (nw == 2) f(t, d, std::integral_constant<int, 2>{});
            else if (nw == 4) f(t, d, std::integral_constant<int, 4>{});
            else f(t, d, std::integral_constant<int, most>{});
        };
        if (dp == 32) dim(std::integral_constant<int, 32>{});
        else if (dp == 64) dim(std::integral_constant<int, 64>{});
        else dim(std::integral_constant<int, 128>{});
    });
}

}  // namespace

ASME_API int asme_window_attention_fwd(const void* q, const void* k, const void* v, void* out, const int64_t* strides,
                                       const uint8_t* valid, int64_t batch, int64_t heads, int64_t kv_heads,
                                       int64_t seq_len, int64_t head_dim, int64_t window, int64_t sinks, int causal,
                                       float scale, int dtype, void* out_low, float* state, void* stream) {
    ASME_CHECK_ARG(q && k && v && out && strides, "asme_window_attention_fwd: null pointer");
    ASME_CHECK_ARG(dtype_ok(dtype), "asme_window_attention_fwd: dtype is 0 (fp32) or 1 (bf16)");
    ASME_CHECK_ARG(sizes_ok(batch, heads, kv_heads, seq_len, head_dim, window, sinks),
                   "asme_window_attention_fwd: bad size");
    ASME_CHECK_ARG(scale > 0.f && scale < INFINITY, "asme_window_attention_fwd: scale > 0");
    Args a = make_args(batch, heads, kv_heads, seq_len, head_dim, window, sinks, causal, scale, valid);
    a.q = tensor(q, strides), a.k = tensor(k, strides + 3), a.v = tensor(v, strides + 6), a.out = tensor(out, strides + 9);
    const int64_t per = 16 / dtype_size(dtype);
    ASME_CHECK_ARG(strides_ok(a.q, per) && strides_ok(a.k, per) && strides_ok(a.v, per) && strides_ok(a.out, per),
                   "asme_window_attention_fwd: 16-byte alignment");
    ASME_CHECK_ARG(!out_low || (dtype == kBF16 && ((uintptr_t)out_low & 15) == 0),
                   "asme_window_attention_fwd: out_low is of bf16, 16-byte aligned");
    a.state = (float2*)state, a.out_low = out_low;
    const int dp = padded_dim(head_dim), nw = waves(batch * heads, seq_len, dtype, dp);
    a.blocks = (int)((seq_len + nw * 32 - 1) / (nw * 32));
    const int64_t items = batch * heads * a.blocks;
    a.items = (uint32_t)items, a.per_xcd = (uint32_t)((items + 7) / 8);
    ASME_CHECK_ARG(items + 8 < (1ll << 31), "asme_window_attention_fwd: bad size");
    with_pass(dtype, dp, nw, [&](auto t, auto d, auto w) {
        hipLaunchKernelGGL((forward_kernel<decltype(t), decltype(d)::value, decltype(w)::value>),
                           dim3((unsigned)(8 * a.per_xcd)), dim3(nw * 64), 0, (hipStream_t)stream, a);
    });
    ASME_LAUNCH_CHECK("asme_window_attention_fwd");
}

// bytes; 0 for sizes that the call refuses
ASME_API int64_t asme_window_attention_bwd_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_len,
                                                     int64_t head_dim, int64_t window, int64_t sinks, int causal,
                                                     int dtype) {
    if (!dtype_ok(dtype) || !sizes_ok(batch, heads, kv_heads, seq_len, head_dim, window, sinks)) return 0;
    Args a = make_args(batch, heads, kv_heads, seq_len, head_dim, window, sinks, causal, 1.f, nullptr);
    plan_kv(a, batch, dtype);
    return ((batch * heads * seq_len + 3) / 4 * 4 + slab_floats(a, batch) + far_floats(a, batch)) * 4;
}

ASME_API int asme_window_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout,
                                       void* dq, void* dk, void* dv, const int64_t* strides, const uint8_t* valid,
                                       int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_len,
                                       int64_t head_dim, int64_t window, int64_t sinks, int causal, float scale,
                                       int dtype, const void* out_low, const float* state, void* workspace,
                                       int64_t ws_bytes, void* stream) {
    ASME_CHECK_ARG(q && k && v && out && dout && dq && dk && dv && strides && state && workspace,
                   "asme_window_attention_bwd: null pointer");
    ASME_CHECK_ARG(dtype_ok(dtype), "asme_window_attention_bwd: dtype is 0 (fp32) or 1 (bf16)");
    ASME_CHECK_ARG(sizes_ok(batch, heads, kv_heads, seq_len, head_dim, window, sinks),
                   "asme_window_attention_bwd: bad size");
    ASME_CHECK_ARG(scale > 0.f && scale < INFINITY, "asme_window_attention_bwd: scale > 0");
    ASME_CHECK_ARG(ws_bytes >= asme_window_attention_bwd_workspace(batch, heads, kv_heads, seq_len, head_dim, window,
                                                                   sinks, causal, dtype) &&
                       ((uintptr_t)workspace & 15) == 0,
                   "asme_window_attention_bwd: workspace too small or not 16-byte aligned");
    Args a = make_args(batch, heads, kv_heads, seq_len, head_dim, window, sinks, causal, scale, valid);
    Tensor* ts[] = {&a.q, &a.k, &a.v, &a.out, &a.dout, &a.dq, &a.dk, &a.dv};
    const void* ps[] = {q, k, v, out, dout, dq, dk, dv};
    const int64_t per = 16 / dtype_size(dtype);
    for (int i = 0; i < 8; ++i) {
        *ts[i] = tensor(ps[i], strides + 3 * i);
        ASME_CHECK_ARG(strides_ok(*ts[i], per), "asme_window_attention_bwd: 16-byte alignment");
    }
    ASME_CHECK_ARG(!out_low || (dtype == kBF16 && ((uintptr_t)out_low & 15) == 0),
                   "asme_window_attention_bwd: out_low is of bf16, 16-byte aligned");
    a.state = (float2*)const_cast<float*>(state), a.out_low = const_cast<void*>(out_low);
    a.delta = (float*)workspace;
    a.part = a.delta + (batch * heads * seq_len + 3) / 4 * 4;
    const int dp = padded_dim(head_dim), nq = waves(batch * heads, seq_len, dtype, dp), nw = waves_kv(seq_len, dtype, dp);
    hipStream_t s = (hipStream_t)stream;
    // the whole grid of `items` workgroups of a pass
    auto grid = [](Args& x, int64_t items) {
        x.items = (uint32_t)items, x.per_xcd = (uint32_t)((items + 7) / 8);
        return dim3(8 * x.per_xcd);
    };
    const int64_t key_heads = batch * kv_heads;
    Args aq = a;
    aq.blocks = (int)((seq_len + nq * 32 - 1) / (nq * 32));
    plan_kv(a, batch, dtype);
    a.far_part = a.part + slab_floats(a, batch);
    const int64_t q_items = batch * heads * aq.blocks, k_items = key_heads * a.blocks * a.near_pieces;
    ASME_CHECK_ARG(q_items + 8 < (1ll << 31) && k_items + 8 < (1ll << 31) &&
                       key_heads * std::max(1, a.far_groups) * a.far_pieces + 8 < (1ll << 31),
                   "asme_window_attention_bwd: bad size");
    const dim3 q_grid = grid(aq, q_items);
    with_pass(dtype, dp, nq, [&](auto t, auto d, auto w) {
        hipLaunchKernelGGL((dq_kernel<decltype(t), decltype(d)::value, decltype(w)::value>), q_grid, dim3(nq * 64), 0, s,
                           aq);
    });
    if (a.far_groups) {
        const dim3 g = grid(a, key_heads * a.far_groups * a.far_pieces);
        with_pass(dtype, dp, kFarWaves, [&](auto t, auto d, auto) {
            hipLaunchKernelGGL((dkv_kernel<decltype(t), decltype(d)::value, kFarWaves, true>), g, dim3(kFarWaves * 64), 0,
                               s, a);
        });
        const int64_t total = key_heads * a.far_groups * 2 * kFarRows * (head_dim / 4);
        hipLaunchKernelGGL(add_far_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, s, a.far_part,
                           a.far_pieces, (int)head_dim, total);
    }
    const dim3 g = grid(a, k_items);
    with_pass(dtype, dp, nw, [&](auto t, auto d, auto w) {
        constexpr int NW = decltype(w)::value == 2 ? 4 : decltype(w)::value;
        hipLaunchKernelGGL((dkv_kernel<decltype(t), decltype(d)::value, NW, false>), g, dim3(nw * 64), 0, s, a);
    });
    if (a.near_pieces > 1) {
        const int64_t total = key_heads * 2 * seq_len * (head_dim / 4);
        with_dtype(dtype, [&](auto t) {
            hipLaunchKernelGGL(add_pieces_kernel<decltype(t)>, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, s, a,
                               total);
        });
    }
    ASME_LAUNCH_CHECK("asme_window_attention_bwd");
}
