// Attention with a learned relative position bias by buckets: kernel arguments and kernels, instantiated per element
// type in bias_attention_{f32,bf16,f16}.hip and launched from bias_attention.hip.
//
//   s_ij = scale q_i.k_j + table[bucket(j - p_i), head],  p_i = offset_b + i,   P = softmax_j(s),   O = P V
//   dS = P o (dO V^T - rowsum(O o dO)),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,
//   dtable[bucket, head] = sum of dS over the pairs of the bucket
//
// Operands.  Every product is taken 32x32 at a time with 16 reduction indices per step: v_mfma_f32_32x32x16_{bf16,f16},
// or eight v_mfma_f32_32x32x2_f32, which read the same fragments (lane l: 8 consecutive reduction indices
// 8 (l / 32) + 0..7 of row / column l % 32; the instruction only needs both operands to agree which index sits where).
// The accumulator of a score tile (element e of lane l: row 8 (e / 4) + 4 (l / 32) + e % 4, column l % 32) then is an
// operand of the next product as it stands, if the other operand is stored with the middle two of every four groups of
// four reduction indices exchanged (perm_group): no score ever passes through LDS.
//
// Bias.  For a pair the offset delta = j - p fixes the bucket, on a map of `width` columns together with the class
// [x_j < x_p] (the offset wraps around a row or does not): a tile of queries x keys meets at most rows + columns - 1
// offsets, so the tile's window of biases is looked up once per tile into LDS and read from there per element.
//
// Statistics.  Row maximum and reciprocal row sum are kept apart: as one number (their log-sum-exp) a row of scores
// near the type's lowest value would lose the sum.  A row that sees no key has maximum 0 and reciprocal 0: its output
// and gradients are zero.
#pragma once
#include <float.h>

#include "common.h"

namespace ba {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int BM = 128;     // queries per workgroup of the forward and dQ kernels: 32 per wave
constexpr int BN = 64;      // keys per LDS tile there
constexpr int KB = 128;     // keys per workgroup of the dK / dV kernel: 32 per wave
constexpr int QB = 32;      // queries per LDS tile there

struct Args {               // strides in elements; out, d_out, dq, dk, dv are dense [B, L, heads, D]
    const void *q, *k, *v, *d_out, *table;
    void *out, *out_lo, *dq, *dk, *dv;
    float *stats, *delta, *part;
    const int *cells, *q_offsets, *kv_len;
    const unsigned char* kpm;
    long q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h;
    int B, H, Hkv, G, Lq, Lk, N, width, nb, causal, off_mode, off, table_type;
    float scale, c;         // c = scale * log2 e
    int heads, queries, tiles, splits;      // few_kernel: heads and queries of a tile of 32 rows, tiles, key ranges
    float *few_o, *few_ml;                  // its partial results if splits > 1
};

enum { F32 = 0, BF16 = 1, F16 = 2 };

typedef float f32x16 __attribute__((ext_vector_type(16)));
template <class T> struct Vec {
    typedef T v8 __attribute__((ext_vector_type(8)));
    typedef T v4 __attribute__((ext_vector_type(4)));
    // probabilities become operands times 2^SHIFT: a half float is subnormal from 2^-14 on, and the rows of a thousand
    // keys hold little else; 2^12 of the row's largest still is far from its end
    static constexpr int SHIFT = 0;
    static constexpr int PAD = 16 / sizeof(T);      // LDS rows are padded by 16 bytes: eight lanes' 16-byte reads meet all banks
};
template <> constexpr int Vec<_Float16>::SHIFT = 12;
template <class T> constexpr float up() { return (float)(1 << Vec<T>::SHIFT); }
template <class T> constexpr float down() { return 1.f / (1 << Vec<T>::SHIFT); }

__device__ __forceinline__ void mma(const Vec<__bf16>::v8& a, const Vec<__bf16>::v8& b, f32x16& acc) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(const Vec<_Float16>::v8& a, const Vec<_Float16>::v8& b, f32x16& acc) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(const Vec<float>::v8& a, const Vec<float>::v8& b, f32x16& acc) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0);
}

__device__ __forceinline__ int perm_group(int g) { return (g & ~3) | ((g & 1) << 1) | ((g >> 1) & 1); }
__device__ __forceinline__ int acc_row(int e, int h) { return (e & 3) + 8 * (e >> 2) + 4 * h; }

// accumulator elements 8 s .. 8 s + 7 as an operand: rounded to T (the matrix instructions of the 16-bit types take
// 16-bit operands; probabilities and their gradients are rounded once, products accumulate in 32 bits)
template <class T> __device__ __forceinline__ typename Vec<T>::v8 acc_frag(const f32x16& a, int s) {
    typename Vec<T>::v8 f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)a[8 * s + j];
    return f;
}

// --- one sequence's positions -------------------------------------------------------------------------------------
struct Seq { int len, off; };
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
    Seq s;
    s.len = a.kv_len ? min(max(a.kv_len[b], 0), a.Lk) : a.Lk;
    s.off = a.off_mode == 2 ? s.len - a.Lq : a.off_mode == 1 ? min(max(a.q_offsets[b], -(1 << 24)), 1 << 24) : a.off;
    return s;
}
// The last key a query may see: none (-1) for rows behind the last query and for positions outside of the buckets' range
__device__ __forceinline__ int last_key(const Args& a, const Seq& s, int i) {
    const int p = s.off + i;
    return i >= a.Lq || p < 0 || p >= a.N ? -1 : a.causal ? p : 0x7fffffff;
}
// bit l: key k0 + l is no padding
__device__ __forceinline__ unsigned long long live_keys(const Args& a, const Seq& s, int b, int k0) {
    const int key = k0 + (threadIdx.x & 63);
    bool ok = key < s.len;
    if (ok && a.kpm) ok = a.kpm[(long)b * a.Lk + key] == 0;
    return __ballot(ok);
}

// --- bias ---------------------------------------------------------------------------------------------------------
// log2 e * table[bucket of (offset delta, class cls)][head].  Scores live in the log2 domain; a finite entry stays
// finite there (the type's lowest value as a mask must not turn into -inf, which hides a key altogether).
__device__ __forceinline__ float bias_at(const Args& a, int cls, int delta, int head) {
    const int i = delta + a.N - 1, n = 2 * a.N - 1;
    if ((unsigned)i >= (unsigned)n) return 0.f;
    const int bucket = a.cells[cls * n + i];
    if ((unsigned)bucket >= (unsigned)a.nb) return 0.f;
    const long at = (long)bucket * a.H + head;
    const float t = a.table_type == F32 ? static_cast<const float*>(a.table)[at]
                  : a.table_type == BF16 ? (float)static_cast<const __bf16*>(a.table)[at]
                                         : (float)static_cast<const _Float16*>(a.table)[at];
    const float r = t * LOG2E;
    return fabsf(t) <= FLT_MAX ? fminf(fmaxf(r, -FLT_MAX), FLT_MAX) : r;
}

// --- LDS tiles ----------------------------------------------------------------------------------------------------
// ROWS x D elements in blocks of 4 x 4 per thread, stored row-major (pitch D + PAD) and / or transposed (pitch
// ROWS + PAD, groups of four rows in perm_group order).  Rows whose bit in `live` is not set are zero: what padding
// holds (infinities, NaN) does not reach a product.
template <class T, int D, int ROWS> struct Tile {
    typedef typename Vec<T>::v4 v4;
    static constexpr int BLOCKS = ROWS * D / 16, NB = (BLOCKS + 255) / 256;
    static constexpr int RP = D + Vec<T>::PAD, CP = ROWS + Vec<T>::PAD;
    static constexpr int ROW_ELEMS = ROWS * RP, COL_ELEMS = D * CP;
    v4 r[NB][4];
    __device__ __forceinline__ void load(const T* base, long stride, unsigned long long live) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int id = threadIdx.x + 256 * i, dg = id % (D / 4), g = id / (D / 4);
            if (BLOCKS % 256 != 0 && id >= BLOCKS) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = 4 * g + j;
                r[i][j] = v4{};
                if ((live >> row) & 1) r[i][j] = *reinterpret_cast<const v4*>(base + row * stride + 4 * dg);
            }
        }
    }
    __device__ __forceinline__ void rows(T* lds) const {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int id = threadIdx.x + 256 * i, dg = id % (D / 4), g = id / (D / 4);
            if (BLOCKS % 256 != 0 && id >= BLOCKS) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<v4*>(lds + (4 * g + j) * RP + 4 * dg) = r[i][j];
        }
    }
    __device__ __forceinline__ void cols(T* lds) const {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int id = threadIdx.x + 256 * i, dg = id % (D / 4), g = id / (D / 4);
            if (BLOCKS % 256 != 0 && id >= BLOCKS) break;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<v4*>(lds + (4 * dg + j) * CP + 4 * perm_group(g)) = v4{r[i][0][j], r[i][1][j], r[i][2][j], r[i][3][j]};
        }
    }
};
template <class T> __device__ __forceinline__ typename Vec<T>::v8 frag(const T* p) {
    return *reinterpret_cast<const typename Vec<T>::v8*>(p);
}
template <class T> __device__ __forceinline__ typename Vec<T>::v8 frag_or_zero(const T* p, bool ok) {
    typename Vec<T>::v8 z = {};
    return ok ? *reinterpret_cast<const typename Vec<T>::v8*>(p) : z;
}

// Workgroup -> (sequence, key/value head, rest).  Consecutive workgroups go to the eight XCDs in turn; where the number
// of key/value heads allows it, all workgroups that read the same keys and values share one XCD's L2.
__device__ __forceinline__ void place(int units, int per_unit, int& unit, int& rest) {
    const int id = blockIdx.x;
    if (units % 8 == 0) {
        unit = (id >> 3) / per_unit * 8 + (id & 7);
        rest = (id >> 3) % per_unit;
    } else {
        unit = id / per_unit;
        rest = id % per_unit;
    }
}

// --- forward ------------------------------------------------------------------------------------------------------
// One workgroup: 128 queries of one head, 32 per wave; keys stream through LDS in tiles of 64.  Queries sit on the
// lanes (S^T = K Q^T), so running maximum and sum are one number per lane.
template <class T, int D, bool MAP>
__global__ __launch_bounds__(256) void fwd_kernel(const Args a) {
    typedef Tile<T, D, BN> KT;
    __shared__ __attribute__((aligned(16))) T sk[KT::ROW_ELEMS];
    __shared__ __attribute__((aligned(16))) T sv[KT::COL_ELEMS];
    __shared__ float sb[MAP ? 2 : 1][BM + BN];
    __shared__ __attribute__((aligned(16))) int sx[BN];
    const int nq = (a.Lq + BM - 1) / BM;
    int unit, rest;
    place(a.B * a.Hkv, a.G * nq, unit, rest);
    const int b = unit / a.Hkv, kvh = unit % a.Hkv, head = kvh * a.G + rest / nq;
    const int q0 = (a.causal ? nq - 1 - rest % nq : rest % nq) * BM;      // causal: the long rows first
    const int w = threadIdx.x >> 6, l = threadIdx.x & 63, col = l & 31, h = l >> 5;
    const int i = q0 + 32 * w + col;
    const Seq s = sequence(a, b);
    const int last = last_key(a, s, i), p = s.off + i;
    const int px = MAP ? ((p % a.width) + a.width) % a.width : 0;
    const T* kb = static_cast<const T*>(a.k) + b * a.k_b + kvh * a.k_h;
    const T* vb = static_cast<const T*>(a.v) + b * a.v_b + kvh * a.v_h;

    typename Vec<T>::v8 qf[D / 16];
    {
        const T* qr = static_cast<const T*>(a.q) + b * a.q_b + (long)i * a.q_l + head * a.q_h;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) qf[c] = frag_or_zero(qr + 16 * c + 8 * h, i < a.Lq);
    }
    f32x16 o[D / 32];
#pragma unroll
    for (int t = 0; t < D / 32; ++t) o[t] = f32x16{};
    float m = -INFINITY, sum = 0.f;

    const int k_end = a.causal ? min(s.len, s.off + min(q0 + BM, a.Lq)) : s.len;
    for (int k0 = 0; k0 < k_end; k0 += BN) {
        const unsigned long long live = live_keys(a, s, b, k0);
        KT tk, tv;
        tk.load(kb + k0 * a.k_l, a.k_l, live);
        tv.load(vb + k0 * a.v_l, a.v_l, live);
        __syncthreads();
        tk.rows(sk);
        tv.cols(sv);
        const int d0 = k0 - (s.off + q0 + BM - 1);
        for (int t = threadIdx.x; t < BM + BN - 1; t += 256) {
            sb[0][t] = bias_at(a, 0, d0 + t, head);
            if (MAP) sb[MAP ? 1 : 0][t] = bias_at(a, 1, d0 + t, head);
        }
        if (MAP && threadIdx.x < BN) sx[threadIdx.x] = (k0 + threadIdx.x) % a.width;
        __syncthreads();

        f32x16 sc[2] = {f32x16{}, f32x16{}};
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) mma(frag<T>(sk + (32 * u + col) * KT::RP + 16 * c + 8 * h), qf[c], sc[u]);

        const int lane_b = BM - 1 - (32 * w + col) + 4 * h;
        const bool masked = live != ~0ull || __any(last < k0 + BN - 1);
        float mx = m;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = 32 * u + 8 * (e >> 2) + (e & 3);       // + 4 h
                float bias = sb[0][lane_b + j];
                if (MAP && sx[j + 4 * h] < px) bias = sb[MAP ? 1 : 0][lane_b + j];
                sc[u][e] = fmaf(sc[u][e], a.c, bias);
            }
        if (masked) {
            const unsigned long long lv = live >> (4 * h);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = 32 * u + 8 * (e >> 2) + (e & 3);
                    if (!((lv >> j) & 1) || k0 + j + 4 * h > last) sc[u][e] = -INFINITY;
                }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[u][e]);
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float ref = mx == -INFINITY ? 0.f : mx;
        if (__any(mx != m)) {
            const float f = __builtin_amdgcn_exp2f(m - ref);
            sum *= f;
#pragma unroll
            for (int t = 0; t < D / 32; ++t) o[t] *= f;
            m = mx;
        }
        const float low = ref - Vec<T>::SHIFT;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                sc[u][e] = __builtin_amdgcn_exp2f(sc[u][e] - low);
                sum += sc[u][e];
            }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const typename Vec<T>::v8 pf = acc_frag<T>(sc[u], c);
#pragma unroll
                for (int t = 0; t < D / 32; ++t) mma(frag<T>(sv + (32 * t + col) * KT::CP + 32 * u + 16 * c + 8 * h), pf, o[t]);
            }
    }
    sum += __shfl_xor(sum, 32);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (i >= a.Lq) return;
    const long row = ((long)b * a.Lq + i) * a.H + head;
    T* out = static_cast<T*>(a.out) + row * D;
    T* lo = a.out_lo ? static_cast<T*>(a.out_lo) + row * D : nullptr;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            typename Vec<T>::v4 hi, rem;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = o[t][4 * g + e] * inv;
                hi[e] = (T)x;
                rem[e] = (T)(x - (float)hi[e]);
            }
            *reinterpret_cast<typename Vec<T>::v4*>(out + 32 * t + 8 * g + 4 * h) = hi;
            if (lo) *reinterpret_cast<typename Vec<T>::v4*>(lo + 32 * t + 8 * g + 4 * h) = rem;
        }
    if (a.stats && h == 0) {
        float* st = a.stats + (((long)b * a.H + head) * a.Lq + i) * 2;
        st[0] = m == -INFINITY ? 0.f : m;
        st[1] = inv * up<T>();
    }
}

// --- forward for few rows -------------------------------------------------------------------------------------------
// A tile is 32 rows: `heads` query heads of one key/value head for `queries` queries each, so that every key and value
// is read once for all of them (one new token: its heads).  A workgroup's four waves take 32-key tiles in turn and join
// at the end; where the tiles are few the keys are cut in `splits` ranges, one workgroup each, joined by merge_kernel.
// Keys go from memory to operand registers (a lane's row), values through the wave's own LDS, transposed; the next tile
// is in flight while this one is worked on.  No barrier until the end.
constexpr int FT = 32;      // keys per tile
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
struct FewRow { int i, head, last, px, p; bool ok; };
__device__ __forceinline__ FewRow few_row(const Args& a, const Seq& s, int kvh, int tile, int r) {
    // tiles: query blocks, then blocks of 32 heads where a key/value head has more than that
    const int qb = (a.Lq + a.queries - 1) / a.queries, gi = r % a.heads, g = tile / qb * a.heads + gi;
    FewRow f;
    f.i = (tile % qb) * a.queries + r / a.heads;
    f.head = kvh * a.G + g;
    f.ok = r < a.heads * a.queries && f.i < a.Lq && g < a.G;
    f.last = f.ok ? last_key(a, s, f.i) : -1;
    f.p = s.off + f.i;
    f.px = a.width ? ((f.p % a.width) + a.width) % a.width : 0;
    return f;
}
template <class T> __device__ __forceinline__ void few_store(const Args& a, int b, const FewRow& f, int D, int d, const float* x,
                                                             float inv) {
    typename Vec<T>::v4 hi, rem;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float y = x[e] * inv;
        hi[e] = (T)y;
        rem[e] = (T)(y - (float)hi[e]);
    }
    const long at = (((long)b * a.Lq + f.i) * a.H + f.head) * D + d;
    *reinterpret_cast<typename Vec<T>::v4*>(static_cast<T*>(a.out) + at) = hi;
    if (a.out_lo) *reinterpret_cast<typename Vec<T>::v4*>(static_cast<T*>(a.out_lo) + at) = rem;
}
template <class T> __device__ __forceinline__ void few_stats(const Args& a, int b, const FewRow& f, float m, float inv) {
    float* st = a.stats + (((long)b * a.H + f.head) * a.Lq + f.i) * 2;
    st[0] = m == -INFINITY ? 0.f : m;
    st[1] = inv * up<T>();
}

template <class T, int D> struct FewLds {
    static constexpr int CP = FT + Vec<T>::PAD, V = D * CP;                              // elements of a wave's values
    static constexpr int JOIN = 4 * 32 * 33 * 4 + 4 * 32 * 2 * 4;                        // bytes of the waves' join
    static constexpr int BYTES = 4 * V * (int)sizeof(T) > JOIN ? 4 * V * (int)sizeof(T) : JOIN;
};
// floats of a wave's bias window, per class
__host__ __device__ __forceinline__ int few_window(int heads, int queries) { return heads * (FT - 1 + queries); }

template <class T, int D, bool MAP>
__global__ __launch_bounds__(256) void few_kernel(const Args a) {
    typedef FewLds<T, D> L;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int unit, rest;
    place(a.B * a.Hkv, a.tiles * a.splits, unit, rest);
    const int b = unit / a.Hkv, kvh = unit % a.Hkv, tile = rest / a.splits, split = rest % a.splits;
    const int w = threadIdx.x >> 6, l = threadIdx.x & 63, col = l & 31, h = l >> 5;
    const Seq s = sequence(a, b);
    const FewRow f = few_row(a, s, kvh, tile, col);
    T* sv = reinterpret_cast<T*>(lds) + w * L::V;
    const int per = FT - 1 + a.queries, window = a.heads * per;
    float* win = reinterpret_cast<float*>(lds + L::BYTES) + w * window * (MAP ? 2 : 1);
    const int i0 = (tile % ((a.Lq + a.queries - 1) / a.queries)) * a.queries, g0 = f.head - kvh * a.G - col % a.heads;
    const T* kb = static_cast<const T*>(a.k) + b * a.k_b + kvh * a.k_h;
    const T* vb = static_cast<const T*>(a.v) + b * a.v_b + kvh * a.v_h;

    typename Vec<T>::v8 qf[D / 16], kf[D / 16];
    {
        const T* qr = static_cast<const T*>(a.q) + b * a.q_b + (long)f.i * a.q_l + f.head * a.q_h;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) qf[c] = frag_or_zero(qr + 16 * c + 8 * h, f.ok);
    }
    f32x16 o[D / 32];
#pragma unroll
    for (int t = 0; t < D / 32; ++t) o[t] = f32x16{};
    float m = -INFINITY, sum = 0.f;

    int end = a.causal ? min(s.len, s.off + min(i0 + a.queries, a.Lq)) : s.len;
    const int all = (max(end, 0) + FT - 1) / FT;
    const int t_begin = (int)((long)all * split / a.splits), t_end = (int)((long)all * (split + 1) / a.splits);

    typename Vec<T>::v4 vr[D / 32][4];
    unsigned live = 0, next_live = 0;
    auto load = [&](int t) {
        const int k0 = t * FT;
        const int key = k0 + col;
        bool ok = t < t_end && key < s.len;
        if (ok && a.kpm) ok = a.kpm[(long)b * a.Lk + key] == 0;
        next_live = (unsigned)__ballot(ok);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) kf[c] = frag_or_zero(kb + key * a.k_l + 16 * c + 8 * h, ok);
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
            const int id = l + 64 * x, dg = id % (D / 4), g = id / (D / 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                vr[x][j] = typename Vec<T>::v4{};
                if ((next_live >> (4 * g + j)) & 1)
                    vr[x][j] = *reinterpret_cast<const typename Vec<T>::v4*>(vb + (long)(k0 + 4 * g + j) * a.v_l + 4 * dg);
            }
        }
    };
    load(t_begin + w);
    for (int t = t_begin + w; t < t_end; t += 4) {
        const int k0 = t * FT;
        live = next_live;
        // offsets of a head's window: key - query from k0 - (p0 + queries - 1) on
        for (int z = l; z < window; z += 64) {
            const int gi = z / per, d = k0 - (s.off + i0 + a.queries - 1) + z % per, head = min(kvh * a.G + g0 + gi, a.H - 1);
            win[z] = bias_at(a, 0, d, head);
            if (MAP) win[window + z] = bias_at(a, 1, d, head);
        }
        f32x16 sc = {};
#pragma unroll
        for (int c = 0; c < D / 16; ++c) mma(kf[c], qf[c], sc);
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
            const int id = l + 64 * x, dg = id % (D / 4), g = id / (D / 4);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<typename Vec<T>::v4*>(sv + (4 * dg + j) * L::CP + 4 * perm_group(g)) =
                    typename Vec<T>::v4{vr[x][0][j], vr[x][1][j], vr[x][2][j], vr[x][3][j]};
        }
        load(t + 4);
        wave_fence();
        const int at = (col % a.heads) * per + a.queries - 1 - col / a.heads + 4 * h;     // rows past the last have no key
        const unsigned lv = live >> (4 * h);
        float mx = m;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int j = 8 * (e >> 2) + (e & 3), key = k0 + j + 4 * h;
            float bias = 0.f;
            if (f.ok) {
                bias = win[at + j];
                if (MAP && key % a.width < f.px) bias = win[window + at + j];
            }
            sc[e] = ((lv >> j) & 1) && key <= f.last ? fmaf(sc[e], a.c, bias) : -INFINITY;
            mx = fmaxf(mx, sc[e]);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float ref = mx == -INFINITY ? 0.f : mx;
        if (__any(mx != m)) {
            const float x = __builtin_amdgcn_exp2f(m - ref);
            sum *= x;
#pragma unroll
            for (int u = 0; u < D / 32; ++u) o[u] *= x;
            m = mx;
        }
        const float low = ref - Vec<T>::SHIFT;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sc[e] = __builtin_amdgcn_exp2f(sc[e] - low);
            sum += sc[e];
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const typename Vec<T>::v8 pf = acc_frag<T>(sc, c);
#pragma unroll
            for (int u = 0; u < D / 32; ++u) mma(frag<T>(sv + (32 * u + col) * L::CP + 16 * c + 8 * h), pf, o[u]);
        }
        wave_fence();
    }
    sum += __shfl_xor(sum, 32);

    // the four waves' results: [wave][channel][row] and (m, sum) [wave][row]
    __syncthreads();
    float* red = reinterpret_cast<float*>(lds);
    float* ml = red + 4 * 32 * 33;
    if (h == 0) {
        ml[(w * 32 + col) * 2] = m;
        ml[(w * 32 + col) * 2 + 1] = sum;
    }
    __syncthreads();
    const int r = threadIdx.x & 31, d4 = (threadIdx.x >> 5) * 4;
    auto joint = [&](int row, float& top, float& total) {
        top = fmaxf(fmaxf(ml[row * 2], ml[(32 + row) * 2]), fmaxf(ml[(64 + row) * 2], ml[(96 + row) * 2]));
        const float ref = top == -INFINITY ? 0.f : top;
        total = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) total += ml[(32 * x + row) * 2 + 1] * __builtin_amdgcn_exp2f(ml[(32 * x + row) * 2] - ref);
        return ref;
    };
    float top, total;
    const float mine = __builtin_amdgcn_exp2f(m - joint(col, top, total));
    joint(r, top, total);
    const FewRow fr = few_row(a, s, kvh, tile, r);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const long part = ((long)unit * a.tiles + tile) * a.splits + split;
#pragma unroll
    for (int u = 0; u < D / 32; ++u) {
#pragma unroll
        for (int e = 0; e < 16; ++e) red[(w * 32 + acc_row(e, h)) * 33 + col] = o[u][e] * mine;
        __syncthreads();
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            x[e] = (red[(d4 + e) * 33 + r] + red[(32 + d4 + e) * 33 + r]) + (red[(64 + d4 + e) * 33 + r] + red[(96 + d4 + e) * 33 + r]);
        if (fr.ok) {
            if (a.splits == 1) few_store<T>(a, b, fr, D, 32 * u + d4, x, inv);
            else *reinterpret_cast<float4*>(a.few_o + (part * 32 + r) * D + 32 * u + d4) = make_float4(x[0], x[1], x[2], x[3]);
        }
        __syncthreads();
    }
    if (fr.ok && d4 == 0) {
        if (a.splits > 1) {
            a.few_ml[(part * 32 + r) * 2] = top;
            a.few_ml[(part * 32 + r) * 2 + 1] = total;
        } else if (a.stats) {
            few_stats<T>(a, b, fr, top, inv);
        }
    }
}

// One workgroup per tile: eight threads a row, the ranges in their order.
template <class T, int D> __global__ __launch_bounds__(256) void merge_kernel(const Args a) {
    const int unit = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles, b = unit / a.Hkv, kvh = unit % a.Hkv;
    const int r = threadIdx.x >> 3, d0 = (threadIdx.x & 7) * (D / 8);
    const Seq s = sequence(a, b);
    const FewRow f = few_row(a, s, kvh, tile, r);
    if (!f.ok) return;
    const long part = ((long)unit * a.tiles + tile) * a.splits;
    float top = -INFINITY, total = 0.f, x[D / 8];
    for (int z = 0; z < a.splits; ++z) top = fmaxf(top, a.few_ml[((part + z) * 32 + r) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int e = 0; e < D / 8; ++e) x[e] = 0.f;
    for (int z = 0; z < a.splits; ++z) {
        const long at = (part + z) * 32 + r;
        const float y = __builtin_amdgcn_exp2f(a.few_ml[at * 2] - ref);
        total += a.few_ml[at * 2 + 1] * y;
#pragma unroll
        for (int e = 0; e < D / 8; e += 4) {
            const float4 v = *reinterpret_cast<const float4*>(a.few_o + at * D + d0 + e);
            x[e] += v.x * y; x[e + 1] += v.y * y; x[e + 2] += v.z * y; x[e + 3] += v.w * y;
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int e = 0; e < D / 8; e += 4) few_store<T>(a, b, f, D, d0 + e, x + e, inv);
    if (a.stats && d0 == 0) few_stats<T>(a, b, f, top, inv);
}

// --- dQ and the sums along the offsets ------------------------------------------------------------------------------
// The forward's split.  A wave adds dS into its own LDS window of offsets, one window per half of the wave: in one
// instruction a half's 32 lanes hold 32 queries and one key, i.e. 32 different offsets, so no two lanes meet and the
// sums have one order.  After each key tile the windows join the workgroup's running sums in wave order; offsets that
// no later tile meets are written out.
template <class T, int D, bool MAP>
__global__ __launch_bounds__(256) void dq_kernel(const Args a) {
    typedef Tile<T, D, BN> KT;
    constexpr int CLS = MAP ? 2 : 1;
    __shared__ __attribute__((aligned(16))) T sk[KT::ROW_ELEMS];
    __shared__ __attribute__((aligned(16))) T skt[KT::COL_ELEMS];
    __shared__ __attribute__((aligned(16))) T sv[KT::ROW_ELEMS];
    __shared__ float sb[CLS][BM + BN];
    __shared__ __attribute__((aligned(16))) int sx[BN];
    __shared__ float win[4][2][CLS][96];
    __shared__ float ring[CLS][256];
    const int nq = (a.Lq + BM - 1) / BM;
    int unit, rest;
    place(a.B * a.Hkv, a.G * nq, unit, rest);
    const int b = unit / a.Hkv, kvh = unit % a.Hkv, head = kvh * a.G + rest / nq;
    const int qblk = a.causal ? nq - 1 - rest % nq : rest % nq, q0 = qblk * BM;
    const int w = threadIdx.x >> 6, l = threadIdx.x & 63, col = l & 31, h = l >> 5;
    const int i = q0 + 32 * w + col;
    const Seq s = sequence(a, b);
    const int last = last_key(a, s, i), p = s.off + i;
    const int px = MAP ? ((p % a.width) + a.width) % a.width : 0;
    const T* kb = static_cast<const T*>(a.k) + b * a.k_b + kvh * a.k_h;
    const T* vb = static_cast<const T*>(a.v) + b * a.v_b + kvh * a.v_h;
    const bool want = a.part != nullptr;

    typename Vec<T>::v8 qf[D / 16], gf[D / 16];
    float m = 0.f, inv = 0.f, delta = 0.f;
    {
        const bool ok = i < a.Lq;
        const T* qr = static_cast<const T*>(a.q) + b * a.q_b + (long)i * a.q_l + head * a.q_h;
        const long row = (((long)b * a.Lq + i) * a.H + head) * D;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            qf[c] = frag_or_zero(qr + 16 * c + 8 * h, ok);
            gf[c] = frag_or_zero(static_cast<const T*>(a.d_out) + row + 16 * c + 8 * h, ok);
            const typename Vec<T>::v8 of = frag_or_zero(static_cast<const T*>(a.out) + row + 16 * c + 8 * h, ok);
#pragma unroll
            for (int j = 0; j < 8; ++j) delta = fmaf((float)of[j], (float)gf[c][j], delta);
            if (a.out_lo) {
                const typename Vec<T>::v8 lf = frag_or_zero(static_cast<const T*>(a.out_lo) + row + 16 * c + 8 * h, ok);
#pragma unroll
                for (int j = 0; j < 8; ++j) delta = fmaf((float)lf[j], (float)gf[c][j], delta);
            }
        }
        delta += __shfl_xor(delta, 32);
        const long st = ((long)b * a.H + head) * a.Lq + i;
        if (ok) {
            m = a.stats[2 * st];
            inv = a.stats[2 * st + 1];
            if (h == 0) a.delta[st] = delta;
        }
    }
    f32x16 dq[D / 32];
#pragma unroll
    for (int t = 0; t < D / 32; ++t) dq[t] = f32x16{};
    if (want) {
        for (int t = threadIdx.x; t < 4 * 2 * CLS * 96; t += 256) (&win[0][0][0][0])[t] = 0.f;
        for (int t = threadIdx.x; t < CLS * 256; t += 256) (&ring[0][0])[t] = 0.f;
    }
    const int span = a.Lk + BM;                 // offsets of a workgroup, as a = j + BM - 1 - (query in workgroup)
    float* part = want ? a.part + (((long)b * a.H + head) * nq + qblk) * CLS * span : nullptr;
    int flushed = 0;

    const int k_end = a.causal ? min(s.len, s.off + min(q0 + BM, a.Lq)) : s.len;
    for (int k0 = 0; k0 < k_end; k0 += BN) {
        const unsigned long long live = live_keys(a, s, b, k0);
        KT tk, tv;
        tk.load(kb + k0 * a.k_l, a.k_l, live);
        tv.load(vb + k0 * a.v_l, a.v_l, live);
        __syncthreads();
        tk.rows(sk);
        tk.cols(skt);
        tv.rows(sv);
        const int d0 = k0 - (s.off + q0 + BM - 1);
        for (int t = threadIdx.x; t < BM + BN - 1; t += 256) {
            sb[0][t] = bias_at(a, 0, d0 + t, head);
            if (MAP) sb[CLS - 1][t] = bias_at(a, 1, d0 + t, head);
        }
        if (MAP && threadIdx.x < BN) sx[threadIdx.x] = (k0 + threadIdx.x) % a.width;
        __syncthreads();

        const int lane_b = BM - 1 - (32 * w + col) + 4 * h;
        const unsigned long long lv = live >> (4 * h);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f32x16 sc = {}, dp = {};
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                mma(frag<T>(sk + (32 * u + col) * KT::RP + 16 * c + 8 * h), qf[c], sc);
                mma(frag<T>(sv + (32 * u + col) * KT::RP + 16 * c + 8 * h), gf[c], dp);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = 32 * u + 8 * (e >> 2) + (e & 3);
                const bool far = MAP && sx[j + 4 * h] < px;
                const float bias = sb[far ? CLS - 1 : 0][lane_b + j];
                float pr = __builtin_amdgcn_exp2f(fmaf(sc[e], a.c, bias) - m) * inv;
                if (!((lv >> j) & 1) || k0 + j + 4 * h > last) pr = 0.f;
                dp[e] = pr * (dp[e] - delta);
                if (want) atomicAdd(&win[w][h][far ? CLS - 1 : 0][j + 4 * h - col + 31], dp[e]);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const typename Vec<T>::v8 df = acc_frag<T>(dp, c);
#pragma unroll
                for (int t = 0; t < D / 32; ++t) mma(frag<T>(skt + (32 * t + col) * KT::CP + 32 * u + 16 * c + 8 * h), df, dq[t]);
            }
        }
        if (want) {
            __syncthreads();
            const int t = threadIdx.x;
            if (t < BM + BN - 1) {
#pragma unroll
                for (int cls = 0; cls < CLS; ++cls) {
                    float add = 0.f;
#pragma unroll
                    for (int ww = 0; ww < 4; ++ww) {
                        const int at = t - 96 + 32 * ww;
                        if (at >= 0 && at < 95) {
                            add += win[ww][0][cls][at] + win[ww][1][cls][at];
                        }
                    }
                    const int slot = (k0 + t) & 255;
                    const float r = ring[cls][slot] + add;
                    if (t < BN) {
                        part[(long)cls * span + k0 + t] = r;
                        ring[cls][slot] = 0.f;
                    } else {
                        ring[cls][slot] = r;
                    }
                }
            }
            __syncthreads();
            for (int z = threadIdx.x; z < 4 * 2 * CLS * 96; z += 256) (&win[0][0][0][0])[z] = 0.f;
            flushed = k0 + BN;
        }
    }
    if (want) {
        __syncthreads();
        for (int t = flushed + threadIdx.x; t < span; t += 256)
#pragma unroll
            for (int cls = 0; cls < CLS; ++cls) part[(long)cls * span + t] = t < flushed + BM - 1 ? ring[cls][t & 255] : 0.f;
    }
    if (i >= a.Lq) return;
    T* out = static_cast<T*>(a.dq) + (((long)b * a.Lq + i) * a.H + head) * D;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            typename Vec<T>::v4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (T)(dq[t][4 * g + e] * a.scale);
            *reinterpret_cast<typename Vec<T>::v4*>(out + 32 * t + 8 * g + 4 * h) = x;
        }
}

// --- dK, dV ---------------------------------------------------------------------------------------------------------
// One workgroup: 128 keys of one key/value head, 32 per wave, their K and V held in registers; the queries of all heads
// that share it stream through LDS, so the sums over those heads stay in the accumulators (no atomics, one order).
// Keys sit on the lanes (S = Q K^T), P and dS are the operands of dV^T = dO^T P and dK^T = Q^T dS as they stand.
template <class T, int D, bool MAP>
__global__ __launch_bounds__(256) void dkv_kernel(const Args a) {
    typedef Tile<T, D, QB> QT;
    __shared__ __attribute__((aligned(16))) T sq[QT::ROW_ELEMS];
    __shared__ __attribute__((aligned(16))) T sqt[QT::COL_ELEMS];
    __shared__ __attribute__((aligned(16))) T sg[QT::ROW_ELEMS];
    __shared__ __attribute__((aligned(16))) T sgt[QT::COL_ELEMS];
    __shared__ float sb[MAP ? 2 : 1][KB + QB];
    __shared__ __attribute__((aligned(16))) float sm[QB], si[QB], sd[QB];
    __shared__ __attribute__((aligned(16))) int sl[QB], sx[QB];
    const int nk = (a.Lk + KB - 1) / KB;
    int unit, rest;
    place(a.B * a.Hkv, nk, unit, rest);
    const int b = unit / a.Hkv, kvh = unit % a.Hkv, k0 = rest * KB;
    const int w = threadIdx.x >> 6, l = threadIdx.x & 63, col = l & 31, h = l >> 5;
    const Seq s = sequence(a, b);
    const int key = k0 + 32 * w + col;
    const bool alive = key < s.len && !(a.kpm && a.kpm[(long)b * a.Lk + key]);
    const int kx = MAP ? key % a.width : 0;

    typename Vec<T>::v8 kf[D / 16], vf[D / 16];
    {
        const T* kr = static_cast<const T*>(a.k) + b * a.k_b + kvh * a.k_h + (long)key * a.k_l;
        const T* vr = static_cast<const T*>(a.v) + b * a.v_b + kvh * a.v_h + (long)key * a.v_l;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            kf[c] = frag_or_zero(kr + 16 * c + 8 * h, alive);
            vf[c] = frag_or_zero(vr + 16 * c + 8 * h, alive);
        }
    }
    f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
    for (int t = 0; t < D / 32; ++t) dk[t] = dv[t] = f32x16{};

    const int i_begin = k0 >= s.len ? a.Lq : a.causal ? max(0, (k0 - s.off) / QB * QB) : 0;
    for (int g = 0; g < a.G; ++g) {
        const int head = kvh * a.G + g;
        const T* qb = static_cast<const T*>(a.q) + b * a.q_b + head * a.q_h;
        const T* gb = static_cast<const T*>(a.d_out) + ((long)b * a.Lq * a.H + head) * D;
        for (int i0 = i_begin; i0 < a.Lq; i0 += QB) {
            const unsigned long long rows = a.Lq - i0 >= QB ? 0xffffffffull : (1ull << (a.Lq - i0)) - 1;
            QT tq, tg;
            tq.load(qb + (long)i0 * a.q_l, a.q_l, rows);
            tg.load(gb + (long)i0 * a.H * D, (long)a.H * D, rows);
            __syncthreads();
            tq.rows(sq);
            tq.cols(sqt);
            tg.rows(sg);
            tg.cols(sgt);
            const int d0 = k0 - (s.off + i0 + QB - 1);
            for (int t = threadIdx.x; t < KB + QB - 1; t += 256) {
                sb[0][t] = bias_at(a, 0, d0 + t, head);
                if (MAP) sb[MAP ? 1 : 0][t] = bias_at(a, 1, d0 + t, head);
            }
            if (threadIdx.x < QB) {
                const int t = threadIdx.x, i = i0 + t, p = s.off + i;
                const long st = ((long)b * a.H + head) * a.Lq + i;
                const bool ok = i < a.Lq;
                sm[t] = ok ? a.stats[2 * st] : 0.f;
                si[t] = ok ? a.stats[2 * st + 1] * up<T>() : 0.f;
                sd[t] = ok ? a.delta[st] * down<T>() : 0.f;
                sl[t] = last_key(a, s, i);
                if (MAP) sx[t] = ((p % a.width) + a.width) % a.width;
            }
            __syncthreads();

            f32x16 sc = {}, dp = {};
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                mma(frag<T>(sq + col * QT::RP + 16 * c + 8 * h), kf[c], sc);
                mma(frag<T>(sg + col * QT::RP + 16 * c + 8 * h), vf[c], dp);
            }
            const int lane_b = 32 * w + col + QB - 1 - 4 * h;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = 8 * (e >> 2) + (e & 3), r = j + 4 * h;
                const bool far = MAP && kx < sx[r];
                const float bias = sb[far && MAP ? 1 : 0][lane_b - j];
                float pr = __builtin_amdgcn_exp2f(fmaf(sc[e], a.c, bias) - sm[r]) * si[r];
                if (!alive || key > sl[r]) pr = 0.f;
                sc[e] = pr;
                dp[e] = pr * fmaf(dp[e], down<T>(), -sd[r]);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const typename Vec<T>::v8 pf = acc_frag<T>(sc, c), df = acc_frag<T>(dp, c);
#pragma unroll
                for (int t = 0; t < D / 32; ++t) {
                    mma(frag<T>(sgt + (32 * t + col) * QT::CP + 16 * c + 8 * h), pf, dv[t]);
                    mma(frag<T>(sqt + (32 * t + col) * QT::CP + 16 * c + 8 * h), df, dk[t]);
                }
            }
        }
    }
    if (key >= a.Lk) return;
    const long row = (((long)b * a.Lk + key) * a.Hkv + kvh) * D;
    T* ok = static_cast<T*>(a.dk) + row;
    T* ov = static_cast<T*>(a.dv) + row;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            typename Vec<T>::v4 x, y;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = (T)(dk[t][4 * g + e] * a.scale);
                y[e] = (T)(dv[t][4 * g + e] * down<T>());
            }
            *reinterpret_cast<typename Vec<T>::v4*>(ok + 32 * t + 8 * g + 4 * h) = x;
            *reinterpret_cast<typename Vec<T>::v4*>(ov + 32 * t + 8 * g + 4 * h) = y;
        }
}

// What the host part launches, one set per element type.
enum { FWD, FEW, MERGE, DQ, DKV };
int launch_f32(int what, int D, const Args& a, unsigned grid, hipStream_t stream);
int launch_bf16(int what, int D, const Args& a, unsigned grid, hipStream_t stream);
int launch_f16(int what, int D, const Args& a, unsigned grid, hipStream_t stream);

template <class T, int D, bool MAP> void launch_one(int what, const Args& a, unsigned grid, hipStream_t stream) {
    if (what == FWD) fwd_kernel<T, D, MAP><<<grid, 256, 0, stream>>>(a);
    else if (what == FEW)
        few_kernel<T, D, MAP><<<grid, 256, FewLds<T, D>::BYTES + 16 * few_window(a.heads, a.queries) * (MAP ? 2 : 1), stream>>>(a);
    else if (what == MERGE) merge_kernel<T, D><<<grid, 256, 0, stream>>>(a);
    else if (what == DQ) dq_kernel<T, D, MAP><<<grid, 256, 0, stream>>>(a);
    else dkv_kernel<T, D, MAP><<<grid, 256, 0, stream>>>(a);
}
template <class T> int launch(int what, int D, const Args& a, unsigned grid, hipStream_t stream) {
    if (D == 32) a.width ? launch_one<T, 32, true>(what, a, grid, stream) : launch_one<T, 32, false>(what, a, grid, stream);
    else if (D == 64) a.width ? launch_one<T, 64, true>(what, a, grid, stream) : launch_one<T, 64, false>(what, a, grid, stream);
    else a.width ? launch_one<T, 128, true>(what, a, grid, stream) : launch_one<T, 128, false>(what, a, grid, stream);
    SPOT_CHECK_LAUNCH("spot_bias_attention");
    return SPOT_OK;
}

}  // namespace ba
