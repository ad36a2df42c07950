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
// MFMAs (common.h, bf16x6); bf16 tensors take one, P and dS rounded to bf16 for their second product (at most 2^-8 of
// each term, the size of the output's own rounding, averaged over the row).  Scores, softmax statistics and all sums are fp32.
#include "elem.h"

using namespace asme;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTS = 64;                  // streamed rows per tile
constexpr int kRowB = 256;               // bytes of a row of an LDS image
constexpr int kImage = kTS * kRowB;      // 16 KiB

typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4;

// the streamed row of accumulator register i in lane half h (32x32 output)
__device__ __forceinline__ int acc_row(int i, int h) { return (i & 3) + 8 * (i >> 2) + 4 * h; }

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
    float2* state;         // (batch, heads, seq_len): maximum of the scaled scores in base 2, 1 / sum
    float* delta;          // (batch, heads, seq_len): D
    float* part;           // partial dK, dV: (key head, split block, piece, 2, rows, dim)
    int seq_len, dim, heads, kv_heads, group, window, sinks, causal;
    int blocks;            // stationary blocks of a sequence
    int64_t items, per_xcd;
    // dK, dV: the first `far_blocks` key blocks hold sinks, which every later query sees: cut into far_pieces pieces;
    // the others into near_pieces
    int far_blocks, far_pieces, near_pieces;
    float scale;
};

// values of 8 columns of a row, on their way to LDS
template <class T>
struct Chunk;
template <>
struct Chunk<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ Frag<3> frag() const {
        const Bf3 s = split_bf3(a, b);
        return {s.h, s.m, s.l};
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
    static_assert(2 * kChunks % kThreads == 0, "whole chunks per thread");
    // two tensors side by side in one image up to 64 columns, in an image each at 128
    static constexpr int kImages = DP == 128 ? 2 : 1;
    static constexpr int kBytes = NP * kImages * kImage;
    using F = Frag<NP>;

    static __device__ __forceinline__ int place(int op, int plane, int row, int ch) {
        if constexpr (DP == 128) return (plane * 2 + op) * kImage + swz(row, ch);
        return plane * kImage + swz(row, ch + op * (DP / 8));
    }
    // bit r: streamed position t0 + r is in the sequence and valid (the same in every wave)
    static __device__ __forceinline__ uint64_t valid_rows(const Args& a, int64_t b, int t0) {
        const int pos = t0 + (threadIdx.x & 63);
        bool ok = pos >= 0 && pos < a.seq_len;
        if (ok && a.valid) ok = a.valid[b * a.seq_len + pos] != 0;
        return __ballot(ok);
    }
    static __device__ __forceinline__ void fetch(Chunk<T> (&c)[kEach], const T* x0, int64_t st0, const T* x1,
                                                 int64_t st1, int t0, uint64_t rows, int dim) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = e * kThreads + threadIdx.x, op = i / kChunks, row = i % kChunks / (DP / 8), ch = i % (DP / 8);
            if (((rows >> row) & 1) && ch * 8 < dim)
                c[e].load((op ? x1 + (t0 + row) * st1 : x0 + (t0 + row) * st0) + ch * 8);
            else
                c[e].zero();
        }
    }
    static __device__ __forceinline__ void put(char* lds, const Chunk<T> (&c)[kEach]) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = e * kThreads + threadIdx.x, op = i / kChunks, row = i % kChunks / (DP / 8), ch = i % (DP / 8);
            const F f = c[e].frag();
#pragma unroll
            for (int p = 0; p < NP; ++p) *reinterpret_cast<bf16x8*>(lds + place(op, p, row, ch)) = f.p[p];
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
    // X[streamed row of the 32-row half `sub`][stationary row] of tensor `op`
    static __device__ __forceinline__ floatx16 score(const char* lds, int op, int sub, const F (&st)[KS]) {
        const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
        floatx16 x;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            F A;
#pragma unroll
            for (int p = 0; p < NP; ++p)
                A.p[p] = *reinterpret_cast<const bf16x8*>(lds + place(op, p, 32 * sub + r32, 2 * ks + h));
            x = product(A, st[ks], x);
        }
        return x;
    }
    // Y^T[feature][stationary row] += streamed^T . x: rows 16 s2 + 8 (j >> 2) + 4 h + (j & 3) of the half are element j of
    // the lane's B fragment; 16-lane group (h, fh) reads rows + q x features 32 ft + 16 fh + 4 p4 .. + 3 transposed
    static __device__ __forceinline__ void gather(const char* lds, int op, int sub, const floatx16& x,
                                                  floatx16 (&y)[NFT]) {
        const int lane = threadIdx.x & 63, h = lane >> 5, fh = (lane >> 4) & 1, q = (lane & 15) >> 2, p4 = lane & 3;
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = x[8 * s2 + j];
            const F P = frag_of(v, (F*)nullptr);
            const int lo = 32 * sub + 16 * s2 + 4 * h + q;
#pragma unroll
            for (int ft = 0; ft < NFT; ++ft) {
                const int ch = 4 * ft + 2 * fh + (p4 >> 1);
                F A;
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_short4*)(lds + place(op, p, lo, ch) + 8 * (p4 & 1)));
                    const short4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_short4*)(lds + place(op, p, lo + 8, ch) + 8 * (p4 & 1)));
                    typedef short short8v __attribute__((ext_vector_type(8)));
                    const short8v c = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                    A.p[p] = __builtin_bit_cast(bf16x8, c);
                }
                y[ft] = product(A, P, y[ft]);
            }
        }
    }
    // row `row` (features 32 ft + 8 i + 4 h .. + 3 of this lane's stationary row) = y * f
    static __device__ __forceinline__ void write_row(T* row, const floatx16 (&y)[NFT], float f, int h, int dim) {
#pragma unroll
        for (int ft = 0; ft < NFT; ++ft)
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
    static __device__ __forceinline__ void clear(floatx16 (&y)[NFT]) {
#pragma unroll
        for (int f = 0; f < NFT; ++f)
#pragma unroll
            for (int i = 0; i < 16; ++i) y[f][i] = 0.f;
    }
};

// Does query i see key j (both valid)?
__device__ __forceinline__ bool sees(const Args& a, int i, int j) {
    const int back = i - j;
    if (a.causal) return back >= 0 && (back < a.window || j < a.sinks);
    return (back < a.window && -back < a.window) || j < a.sinks;
}
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
__device__ __forceinline__ bool item_of(const Args& a, int64_t& item) {
    item = (int64_t)(blockIdx.x % 8) * a.per_xcd + blockIdx.x / 8;
    return item < a.items && (int64_t)(blockIdx.x / 8) < a.per_xcd;
}

// The streamed key tiles of queries [q0, q1): those of the sinks in front of the window's first tile, then the window's.
struct KeyTiles {
    int sink_tiles, lo, count;
    __device__ KeyTiles(const Args& a, int q0, int q1) {
        lo = max(0, q0 - a.window + 1) / kTS * kTS;
        const int hi = a.causal ? q1 : (int)min((int64_t)a.seq_len, (int64_t)q1 - 1 + a.window);
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
    int64_t item;
    if (!item_of(a, item)) return;  // (the whole workgroup)
    const int lane = threadIdx.x & 63, h = lane >> 5, r32 = lane & 31;
    const int block = (int)(item % a.blocks), head = (int)(item / a.blocks % a.heads);
    const int64_t b = item / a.blocks / a.heads;
    const int q0 = block * NW * 32, q1 = min(a.seq_len, q0 + NW * 32);
    const int w0 = q0 + (threadIdx.x >> 6) * 32, qi = w0 + r32;
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
    int i = 0, t0 = 0;
    uint64_t rows = 0;
    auto advance = [&]() {  // the next tile with a valid position, on its way
        for (; i < tiles.count; ++i) {
            t0 = tiles.start(i);
            rows = P::valid_rows(a, b, t0);
            if (rows) break;
        }
        if (i < tiles.count) P::fetch(next, K, a.k.st, V, a.v.st, t0, rows, a.dim);
    };
    if (__syncthreads_or(any)) advance();
    else i = tiles.count;
    while (i < tiles.count) {
        const int k0 = t0;
        const uint64_t keys = rows;
        __syncthreads();  // the last tile has been read
        P::put(lds, next);
        __syncthreads();
        ++i;
        advance();
        if (!any) continue;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const uint32_t ok = (uint32_t)(keys >> (32 * sub));
            const int j0 = k0 + 32 * sub, seen = ok ? block_seen(a, w0, j0) : 0;
            if (!seen) continue;
            floatx16 x = P::score(lds, 0, sub, Q);
            if (seen == 1 || ok != 0xFFFFFFFFu) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int r = acc_row(e, h);
                    x[e] = ((ok >> r) & 1) && sees(a, qi, j0 + r) ? x[e] : -INFINITY;
                }
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
            P::gather(lds, 1, sub, x, y);
        }
    }
    sum += __shfl_xor(sum, 32, 64);
    if (qi >= a.seq_len) return;
    const float inv = live ? 1.f / sum : 0.f;
    if (!live) P::clear(y);
    P::write_row(a.out.at<T>(b, head) + qi * a.out.st, y, inv, h, a.dim);
    // a position that is no query: P = 2^-inf = 0 in the backward
    if (a.state && h == 0) a.state[(b * a.heads + head) * a.seq_len + qi] = make_float2(live ? top : INFINITY, inv);
}

// ------------------------------------------------------------------------------------------------ dQ
template <class T, int DP, int NW>
__global__ __launch_bounds__(NW * 64) void dq_kernel(Args a) {
    using P = Pass<T, DP, NW>;
    __shared__ __attribute__((aligned(16))) char lds[P::kBytes];
    int64_t item;
    if (!item_of(a, item)) return;
    const int lane = threadIdx.x & 63, h = lane >> 5, r32 = lane & 31;
    const int block = (int)(item % a.blocks), head = (int)(item / a.blocks % a.heads);
    const int64_t b = item / a.blocks / a.heads;
    const int q0 = block * NW * 32, q1 = min(a.seq_len, q0 + NW * 32);
    const int w0 = q0 + (threadIdx.x >> 6) * 32, qi = w0 + r32;
    const bool live = qi < a.seq_len && (!a.valid || a.valid[b * a.seq_len + qi]);
    const bool any = __ballot(live) != 0;
    typename P::F Q[P::KS], O[P::KS];
    P::stationary(Q, live ? a.q.at<T>(b, head) + qi * a.q.st : nullptr, h, a.dim);
    P::stationary(O, live ? a.dout.at<T>(b, head) + qi * a.dout.st : nullptr, h, a.dim);
    // D of the row: each half of the lanes holds half of its columns
    float delta = 0.f;
    if (live) {
        const T* o = a.out.at<T>(b, head) + qi * a.out.st;
        const T* d = a.dout.at<T>(b, head) + qi * a.dout.st;
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
    int i = 0, t0 = 0;
    uint64_t rows = 0;
    auto advance = [&]() {
        for (; i < tiles.count; ++i) {
            t0 = tiles.start(i);
            rows = P::valid_rows(a, b, t0);
            if (rows) break;
        }
        if (i < tiles.count) P::fetch(next, K, a.k.st, V, a.v.st, t0, rows, a.dim);
    };
    if (__syncthreads_or(any)) advance();
    else i = tiles.count;
    while (i < tiles.count) {
        const int k0 = t0;
        const uint64_t keys = rows;
        __syncthreads();
        P::put(lds, next);
        __syncthreads();
        ++i;
        advance();
        if (!any) continue;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const uint32_t ok = (uint32_t)(keys >> (32 * sub));
            const int j0 = k0 + 32 * sub, seen = ok ? block_seen(a, w0, j0) : 0;
            if (!seen) continue;
            floatx16 x = P::score(lds, 0, sub, Q);
            const floatx16 dp = P::score(lds, 1, sub, O);
            const bool test = seen == 1 || ok != 0xFFFFFFFFu;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float p = __builtin_amdgcn_exp2f(fmaf(x[e], c, -st.x)) * st.y;
                if (test) {
                    const int r = acc_row(e, h);
                    p = ((ok >> r) & 1) && sees(a, qi, j0 + r) ? p : 0.f;
                }
                x[e] = p * (dp[e] - delta);
            }
            P::gather(lds, 0, sub, x, y);
        }
    }
    if (qi >= a.seq_len) return;
    if (!live) P::clear(y);
    P::write_row(a.dq.at<T>(b, head) + qi * a.dq.st, y, a.scale, h, a.dim);
}

// ------------------------------------------------------------------------------------------------ dK, dV
// Item: (sequence, key head, key block, piece); its steps are the query tiles of the block's range for each query head of
// the group, of which a piece takes a contiguous share.  One piece: dK and dV at once, else partial rows.
template <class T, int DP, int NW>
__global__ __launch_bounds__(NW * 64) void dkv_kernel(Args a) {
    using P = Pass<T, DP, NW>;
    __shared__ __attribute__((aligned(16))) char lds[P::kBytes];
    __shared__ __attribute__((aligned(16))) float meta[3][kTS];  // maximum, 1 / sum, D of the tile's queries
    int64_t item;
    if (!item_of(a, item)) return;
    const int lane = threadIdx.x & 63, h = lane >> 5, r32 = lane & 31;
    const int near = a.blocks - a.far_blocks, per_head = a.far_blocks * a.far_pieces + near * a.near_pieces;
    const int64_t bk = item / per_head, b = bk / a.kv_heads;
    const int kh = (int)(bk % a.kv_heads);
    int within = (int)(item % per_head), block, piece, pieces;
    if (within < a.far_blocks * a.far_pieces) {
        pieces = a.far_pieces, block = within / pieces, piece = within % pieces;
    } else {
        within -= a.far_blocks * a.far_pieces;
        pieces = a.near_pieces, block = a.far_blocks + within / pieces, piece = within % pieces;
    }
    const int k0 = block * NW * 32, k1 = min(a.seq_len, k0 + NW * 32);
    const int w0 = k0 + (threadIdx.x >> 6) * 32, kj = w0 + r32;
    const bool live = kj < a.seq_len && (!a.valid || a.valid[b * a.seq_len + kj]);
    const bool any = __ballot(live) != 0;
    const uint32_t ok = (uint32_t)__ballot(live);  // (both halves of the lanes hold the same keys)
    typename P::F K[P::KS], V[P::KS];
    P::stationary(K, live ? a.k.at<T>(b, kh) + kj * a.k.st : nullptr, h, a.dim);
    P::stationary(V, live ? a.v.at<T>(b, kh) + kj * a.v.st : nullptr, h, a.dim);
    floatx16 yk[P::NFT], yv[P::NFT];
    P::clear(yk);
    P::clear(yv);
    const float c = a.scale * kLog2e;
    // the queries that see a key of the block
    const bool all = k0 < a.sinks;
    const int lo = (a.causal ? k0 : all ? 0 : max(0, k0 - a.window + 1)) / kTS * kTS;
    const int hi = all ? a.seq_len : (int)min((int64_t)a.seq_len, (int64_t)k1 - 1 + a.window);
    const int tiles = (hi - lo + kTS - 1) / kTS, steps = tiles * a.group;
    int i = (int)((int64_t)steps * piece / pieces), t0 = 0, head = 0;
    const int last = (int)((int64_t)steps * (piece + 1) / pieces);
    uint64_t rows = 0;
    Chunk<T> next[P::kEach];
    float2 st = make_float2(INFINITY, 0.f);
    float delta = 0.f;
    auto advance = [&]() {
        for (; i < last; ++i) {
            t0 = lo + i % tiles * kTS;
            rows = P::valid_rows(a, b, t0);
            if (rows) break;
        }
        if (i < last) {
            head = kh * a.group + i / tiles;
            P::fetch(next, a.q.at<T>(b, head), a.q.st, a.dout.at<T>(b, head), a.dout.st, t0, rows, a.dim);
            if (threadIdx.x < kTS) {
                const int64_t at = (b * a.heads + head) * a.seq_len + t0 + threadIdx.x;
                st = make_float2(INFINITY, 0.f), delta = 0.f;
                if ((rows >> threadIdx.x) & 1) st = a.state[at], delta = a.delta[at];
            }
        }
    };
    if (__syncthreads_or(any)) advance();
    else i = last;
    while (i < last) {
        const int q0 = t0;
        const uint64_t queries = rows;
        __syncthreads();
        P::put(lds, next);
        if (threadIdx.x < kTS) meta[0][threadIdx.x] = st.x, meta[1][threadIdx.x] = st.y, meta[2][threadIdx.x] = delta;
        __syncthreads();
        ++i;
        advance();
        if (!any) continue;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int i0 = q0 + 32 * sub, seen = (uint32_t)(queries >> (32 * sub)) ? block_seen(a, i0, w0) : 0;
            if (!seen) continue;
            floatx16 x = P::score(lds, 0, sub, K);
            floatx16 dp = P::score(lds, 1, sub, V);
            const bool test = seen == 1 || ok != 0xFFFFFFFFu;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const floatx4 m = *reinterpret_cast<const floatx4*>(&meta[0][32 * sub + 8 * g + 4 * h]);
                const floatx4 v = *reinterpret_cast<const floatx4*>(&meta[1][32 * sub + 8 * g + 4 * h]);
                const floatx4 d = *reinterpret_cast<const floatx4*>(&meta[2][32 * sub + 8 * g + 4 * h]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float p = __builtin_amdgcn_exp2f(fmaf(x[4 * g + e], c, -m[e])) * v[e];
                    if (test) p = live && sees(a, i0 + 8 * g + 4 * h + e, kj) ? p : 0.f;
                    x[4 * g + e] = p;
                    dp[4 * g + e] = p * (dp[4 * g + e] - d[e]);
                }
            }
            P::gather(lds, 1, sub, x, yv);
            P::gather(lds, 0, sub, dp, yk);
        }
    }
    if (pieces > 1) {  // fp32 rows of this piece, zeros where there is nothing
        const int64_t far = (int64_t)a.far_blocks * (a.far_pieces > 1 ? a.far_pieces : 0);
        const int64_t split = far + (int64_t)near * (a.near_pieces > 1 ? a.near_pieces : 0);
        const int64_t slab = bk * split + (block < a.far_blocks ? (int64_t)block * a.far_pieces
                                                                : far + (int64_t)(block - a.far_blocks) * a.near_pieces) +
                             piece;
        float* p = a.part + (slab * 2 * NW * 32 + (kj - k0)) * a.dim;
        using PF = Pass<float, DP, NW>;
        PF::write_row(p, yk, a.scale, h, a.dim);
        PF::write_row(p + (int64_t)NW * 32 * a.dim, yv, 1.f, h, a.dim);
        return;
    }
    if (kj >= a.seq_len) return;
    if (!live) P::clear(yk), P::clear(yv);
    P::write_row(a.dk.at<T>(b, kh) + kj * a.dk.st, yk, a.scale, h, a.dim);
    P::write_row(a.dv.at<T>(b, kh) + kj * a.dv.st, yv, 1.f, h, a.dim);
}

// dK, dV of the blocks in pieces: their partial rows added in order, 4 columns a thread
template <class T>
__global__ __launch_bounds__(256) void add_pieces_kernel(Args a, int block_rows, int first, int blocks, int pieces,
                                                         int64_t slab0, int64_t slabs, int64_t total) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int quads = a.dim / 4, c = (int)(i % quads) * 4, row = (int)(i / quads % block_rows);
    const int64_t u = i / quads / block_rows;
    const int which = (int)(u % 2), block = (int)(u / 2 % blocks);
    const int64_t bk = u / 2 / blocks, b = bk / a.kv_heads;
    const int kh = (int)(bk % a.kv_heads), kj = (first + block) * block_rows + row;
    if (kj >= a.seq_len) return;
    const bool live = !a.valid || a.valid[b * a.seq_len + kj];
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (live)
        for (int p = 0; p < pieces; ++p) {
            float x[4];
            Elem<float>::load(a.part + (((bk * slabs + slab0 + (int64_t)block * pieces + p) * 2 + which) * block_rows +
                                        row) * a.dim + c, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += x[e];
        }
    const Tensor& t = which ? a.dv : a.dk;
    T* o = t.at<T>(b, kh) + kj * t.st + c;
#pragma unroll
    for (int e = 0; e < 4; ++e) Elem<T>::put(o + e, s[e]);
}

// ------------------------------------------------------------------------------------------------ host
int padded_dim(int64_t dim) { return dim <= 32 ? 32 : (int)dim; }

// waves (of 32 stationary rows) per workgroup
int waves(int64_t seq_len, int dtype, int dp) {
    if (seq_len <= 64) return 2;
    return dtype == kF32 && dp == 128 ? 4 : 8;
}

struct Pieces {
    int far_blocks, far_pieces, near_pieces;
    int64_t slabs;  // partial slabs per key head
};
// key blocks are cut so that none takes much longer than the others: a block with sinks is seen by every later query
Pieces pieces_of(int64_t batch, int64_t kv_heads, int64_t group, int64_t seq_len, int64_t window, int64_t sinks, int nw) {
    const int64_t rows = nw * 32, blocks = (seq_len + rows - 1) / rows;
    Pieces p;
    p.far_blocks = (int)std::min(blocks, (sinks + rows - 1) / rows);
    const int64_t near_steps = std::min(seq_len, rows + window) * group, far_steps = seq_len * group;
    const int64_t have = batch * kv_heads * blocks;
    p.near_pieces = (int)std::max<int64_t>(1, std::min<int64_t>({(512 + have - 1) / have / 2 + (have >= 512 ? 0 : 1),
                                                                  near_steps / 512, 16}));
    if (have >= 256) p.near_pieces = 1;
    p.far_pieces = (int)std::max<int64_t>(
        1, std::min<int64_t>(64, far_steps / std::max<int64_t>(512, near_steps / p.near_pieces)));
    p.slabs = (int64_t)p.far_blocks * (p.far_pieces > 1 ? p.far_pieces : 0) +
              (blocks - p.far_blocks) * (p.near_pieces > 1 ? p.near_pieces : 0);
    return p;
}

bool sizes_ok(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_len, int64_t dim, int64_t window,
              int64_t sinks) {
    return batch >= 1 && kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && seq_len >= 1 &&
           seq_len <= (1 << 24) && (dim == 16 || dim == 32 || dim == 64 || dim == 128) && window >= 1 && sinks >= 0 &&
           heads <= 65536 && batch <= (1ll << 24) && batch * heads * seq_len <= (1ll << 34);
}

bool strides_ok(const Tensor& t, int64_t per) {
    return t.p && ((uintptr_t)t.p & 15) == 0 && t.sb % per == 0 && t.st % per == 0 && t.sh % per == 0;
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
            constexpr bool wide = sizeof(t) == 4 && decltype(d)::value == 128;
            if (nw == 2) f(t, d, std::integral_constant<int, 2>{});
            else f(t, d, std::integral_constant<int, wide ? 4 : 8>{});
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
                                       float scale, int dtype, float* state, void* stream) {
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
    a.state = (float2*)state;
    const int dp = padded_dim(head_dim), nw = waves(seq_len, dtype, dp);
    a.blocks = (int)((seq_len + nw * 32 - 1) / (nw * 32));
    a.items = batch * heads * a.blocks;
    a.per_xcd = (a.items + 7) / 8;
    ASME_CHECK_ARG(8 * a.per_xcd < (1ll << 31), "asme_window_attention_fwd: bad size");
    with_pass(dtype, dp, nw, [&](auto t, auto d, auto w) {
        hipLaunchKernelGGL((forward_kernel<decltype(t), decltype(d)::value, decltype(w)::value>),
                           dim3((unsigned)(8 * a.per_xcd)), dim3(nw * 64), 0, (hipStream_t)stream, a);
    });
    ASME_LAUNCH_CHECK("asme_window_attention_fwd");
}

// bytes; 0 for sizes that the call refuses
ASME_API int64_t asme_window_attention_bwd_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_len,
                                                     int64_t head_dim, int64_t window, int64_t sinks, int dtype) {
    if (!dtype_ok(dtype) || !sizes_ok(batch, heads, kv_heads, seq_len, head_dim, window, sinks)) return 0;
    const int nw = waves(seq_len, dtype, padded_dim(head_dim));
    const Pieces p = pieces_of(batch, kv_heads, heads / kv_heads, seq_len, std::min(window, seq_len),
                               std::min(sinks, seq_len), nw);
    return ((batch * heads * seq_len + 3) / 4 * 4 + batch * kv_heads * p.slabs * 2 * nw * 32 * head_dim) * 4;
}

ASME_API int asme_window_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout,
                                       void* dq, void* dk, void* dv, const int64_t* strides, const uint8_t* valid,
                                       int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_len,
                                       int64_t head_dim, int64_t window, int64_t sinks, int causal, float scale,
                                       int dtype, const float* state, void* workspace, int64_t ws_bytes, void* stream) {
    ASME_CHECK_ARG(q && k && v && out && dout && dq && dk && dv && strides && state && workspace,
                   "asme_window_attention_bwd: null pointer");
    ASME_CHECK_ARG(dtype_ok(dtype), "asme_window_attention_bwd: dtype is 0 (fp32) or 1 (bf16)");
    ASME_CHECK_ARG(sizes_ok(batch, heads, kv_heads, seq_len, head_dim, window, sinks),
                   "asme_window_attention_bwd: bad size");
    ASME_CHECK_ARG(scale > 0.f && scale < INFINITY, "asme_window_attention_bwd: scale > 0");
    ASME_CHECK_ARG(ws_bytes >= asme_window_attention_bwd_workspace(batch, heads, kv_heads, seq_len, head_dim, window,
                                                                   sinks, dtype) &&
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
    a.state = (float2*)const_cast<float*>(state);
    a.delta = (float*)workspace;
    a.part = a.delta + (batch * heads * seq_len + 3) / 4 * 4;
    const int dp = padded_dim(head_dim), nw = waves(seq_len, dtype, dp), rows = nw * 32;
    a.blocks = (int)((seq_len + rows - 1) / rows);
    const Pieces p = pieces_of(batch, kv_heads, a.group, seq_len, a.window, a.sinks, nw);
    a.far_blocks = p.far_blocks, a.far_pieces = p.far_pieces, a.near_pieces = p.near_pieces;
    hipStream_t s = (hipStream_t)stream;
    const int64_t q_items = batch * heads * a.blocks;
    const int64_t k_items = batch * kv_heads * ((int64_t)a.far_blocks * a.far_pieces +
                                                (int64_t)(a.blocks - a.far_blocks) * a.near_pieces);
    ASME_CHECK_ARG(q_items + 8 < (1ll << 31) && k_items + 8 < (1ll << 31), "asme_window_attention_bwd: bad size");
    with_pass(dtype, dp, nw, [&](auto t, auto d, auto w) {
        using T = decltype(t);
        constexpr int DP = decltype(d)::value, NW = decltype(w)::value;
        a.items = q_items, a.per_xcd = (q_items + 7) / 8;
        hipLaunchKernelGGL((dq_kernel<T, DP, NW>), dim3((unsigned)(8 * a.per_xcd)), dim3(nw * 64), 0, s, a);
        a.items = k_items, a.per_xcd = (k_items + 7) / 8;
        hipLaunchKernelGGL((dkv_kernel<T, DP, NW>), dim3((unsigned)(8 * a.per_xcd)), dim3(nw * 64), 0, s, a);
    });
    const int64_t far_slabs = (int64_t)a.far_blocks * (a.far_pieces > 1 ? a.far_pieces : 0);
    auto add = [&](int first, int blocks, int pieces, int64_t slab0) {
        if (blocks <= 0 || pieces <= 1) return;
        const int64_t total = batch * kv_heads * blocks * 2 * rows * (head_dim / 4);
        with_dtype(dtype, [&](auto t) {
            hipLaunchKernelGGL(add_pieces_kernel<decltype(t)>, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, s, a,
                               rows, first, blocks, pieces, slab0, p.slabs, total);
        });
    };
    add(0, a.far_blocks, a.far_pieces, 0);
    add(a.far_blocks, a.blocks - a.far_blocks, a.near_pieces, far_slabs);
    ASME_LAUNCH_CHECK("asme_window_attention_bwd");
}
