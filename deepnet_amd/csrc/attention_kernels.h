// Cross attention on the matrix cores: kernels and their launcher for one element type (attention.hip: single precision and the entry
// points, attention_f64.hip: double precision).
//
// Queries [B; Hq; Lq; Dk], keys [B; Hk; Lk; Dk], values [B; Hk; Lk; Dv], Hq = G Hk: the G query heads of a key head form one list of
// G Lq rows, so keys and values are staged once for all of them and their gradients are summed over the group by construction.
//
//   S = scale q k^T     P = softmax over the keys that the mask [B; Lk] leaves     out = P v     lse = log sum e^S
//   delta = sum_d d_out out    dS = scale P (d_out v^T - delta)    dq = dS k    dk = dS^T q    dv = P^T d_out
//
// Matrix instructions of shape M x M x K: lane l supplies A[l % M][l / M] and B[l / M][l % M] and holds column l % M of the result, in
// register r the row acc_row(r, l / M).  The products are arranged so that nothing is transposed: a wavefront computes S^T (keys down,
// queries across), so the maximum and the sum of a query are over a lane's own registers and its M-distant neighbours, and register r
// of P^T is, as it stands, the B operand of the step of out^T = v^T P^T that runs over the keys { acc_row(r, 0), acc_row(r, 1), ... }.
// The backward pass uses the same property with queries and keys in either role.
#pragma once

#include "model_ops.h"

namespace dnh {

// G lane groups (= K of the instruction), R result registers, N elements of 16 bytes.  Exponentials are taken in the base whose
// logarithm of e is kBase: it goes into the scale.
struct MmaBaseF32 {
    typedef float T;
    static __device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x); }
    static __device__ __forceinline__ float log_(float x) { return __log2f(x); }
    static constexpr double kBase = 1.44269504088896340736;
};
struct MmaF32 : MmaBaseF32 {      // v_mfma_f32_32x32x2_f32
    static constexpr int M = 32, G = 2, R = 16, N = 4;
    typedef float Acc __attribute__((ext_vector_type(16)));
    static __device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }
    static __device__ __forceinline__ Acc mfma(float a, float b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
};
struct MmaF32Few : MmaBaseF32 {   // v_mfma_f32_16x16x4_f32
    static constexpr int M = 16, G = 4, R = 4, N = 4;
    typedef float Acc __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ int acc_row(int r, int h) { return 4 * h + r; }
    static __device__ __forceinline__ Acc mfma(float a, float b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
};
struct MmaF64 {                   // v_mfma_f64_16x16x4_f64
    typedef double T;
    static constexpr int M = 16, G = 4, R = 4, N = 2;
    typedef double Acc __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ int acc_row(int r, int h) { return 4 * r + h; }
    static __device__ __forceinline__ Acc mfma(double a, double b, Acc c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ double exp_(double x) { return exp(x); }
    static __device__ __forceinline__ double log_(double x) { return log(x); }
    static constexpr double kBase = 1.0;
};
template <class T> struct MmaOf;
template <> struct MmaOf<float> {
    typedef MmaF32 Tile;
    typedef MmaF32Few Few;
};
template <> struct MmaOf<double> {
    typedef MmaF64 Tile;
    typedef MmaF64 Few;
};

constexpr int kAttTile = 32;    // keys (forward, dq) or query rows (dk, dv) of one step
constexpr int kAttWords = 256;  // mask words kept in LDS at a time

struct Strides4 {
    int64_t b, h, l, d;
};
template <class T> struct AttArgs {
    const T *q, *k, *v, *out, *d_out;
    T *o, *dq, *dk, *dv;      // o: the forward result
    T* lse_out;               // may be missing
    const T* lse;
    const uint8_t* mask;      // may be missing
    Strides4 sq, sk, sv, so, sdo, sdq, sdk, sdv;   // so: out / o
    Strides4 slse;            // b, h, l
    int64_t mask_b, mask_l;
    int B, Hk, G, Lq, Lk, Dk, Dv;
    uint32_t rows;            // G Lq
    T scale, scale_base;      // scale, and scale x log e in the exponentials' base
    bool vec;                 // q, k, v (and d_out) are contiguous along their last axis
    // workgroups of a key head: row blocks x shares of the keys (forward, dq), key blocks x shares of the rows (dk, dv)
    uint32_t blocks, splits, split_tiles;
    uint32_t kblocks, ksplits, ksplit_tiles;
    T *part_o, *part_m, *part_l;      // forward: a share's unnormalised result, maximum and sum
    T *part_dq, *part_dk, *part_dv;   // backward: a share's sums, [share][head][row or key][width]
    T* delta;
};

// Which (batch, key head) and which of its `per` workgroups number `at` of a range is.  Consecutive workgroups go to the eight XCDs in
// turn: a head stays on one XCD, whose L2 then holds its keys and values, and consecutive heads (which share a sequence, and its length)
// go to different ones.
__device__ __forceinline__ void att_place(uint32_t at, uint32_t per, uint32_t heads, uint32_t* head, uint32_t* inner) {
    const uint32_t full = heads & ~7u;
    if (at < full * per) {
        const uint32_t j = at >> 3, k = j / per;
        *head = (at & 7) + 8 * k;
        *inner = j - k * per;
    } else {
        const uint32_t j = at - full * per, k = j / per;
        *head = full + k;
        *inner = j - k * per;
    }
}

// 16 bytes of a row at element d, zeros beyond D
template <class T>
__device__ __forceinline__ typename Vec16<T>::type att_load(const T* row, int d, int D, int64_t sd, bool vec) {
    using V = typename Vec16<T>::type;
    constexpr int N = kVecN<T>;
    if (vec && d + N <= D) return *(const V*)(row + d);
    V v = 0;
#pragma unroll
    for (int e = 0; e < N; e++)
        if (d + e < D) v[e] = row[(int64_t)(d + e) * sd];
    return v;
}

template <class T, int DP> constexpr int kAttPitch = DP + kVecN<T>;   // LDS rows: 16 rows' 16-byte reads fall on different banks

template <class T> __device__ __forceinline__ bool att_key_on(const AttArgs<T>& p, int b, int key) {
    return key < p.Lk && (!p.mask || p.mask[b * p.mask_b + key * p.mask_l] != 0);
}
// 32-bit words of which keys are attended to, for tiles [t0, t0 + n), n <= kAttWords; the whole workgroup calls it
template <class T>
__device__ __forceinline__ void att_words(const AttArgs<T>& p, int b, int t0, int n, uint32_t* words, int threads) {
    for (int i = threadIdx.x; i < (n * kAttTile + 63) / 64 * 64; i += threads) {
        const unsigned long long m = __ballot(att_key_on(p, b, t0 * kAttTile + i));
        if ((threadIdx.x & 63) == 0) {
            words[i / 32] = (uint32_t)m;
            words[i / 32 + 1] = (uint32_t)(m >> 32);
        }
    }
}

// A tile of 32 rows of two matrices on its way from memory to LDS: loaded into registers while the tile before it is worked on.
template <class T, int DP, int WAVES> struct AttStage {
    using V = typename Vec16<T>::type;
    static constexpr int N = kVecN<T>, PER = DP / N, NL = kAttTile * PER / (64 * WAVES);
    static_assert(NL * 64 * WAVES == kAttTile * PER, "the workgroup covers a tile evenly");
    V a[NL], b[NL];
    // row(r, which): address of row r of the tile (always readable); rows whose bit is not set become zeros
    template <class Row>
    __device__ __forceinline__ void load(Row row, int Da, int Db, int64_t sda, int64_t sdb, bool vec, uint32_t word) {
        const bool whole = vec && Da == DP && Db == DP;
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const int i = threadIdx.x + j * 64 * WAVES, r = i / PER, d = (i - r * PER) * N;
            const T *pa = row(r, 0), *pb = row(r, 1);
            if (whole) {
                a[j] = *(const V*)(pa + d);
                b[j] = *(const V*)(pb + d);
            } else {
                a[j] = att_load<T>(pa, d, Da, sda, vec);
                b[j] = att_load<T>(pb, d, Db, sdb, vec);
            }
        }
        if (word != ~0u) {
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int r = (threadIdx.x + j * 64 * WAVES) / PER;
                if (!((word >> r) & 1u)) a[j] = b[j] = 0;
            }
        }
    }
    __device__ __forceinline__ void store(T* la, T* lb) const {
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const int i = threadIdx.x + j * 64 * WAVES, r = i / PER, d = (i - r * PER) * N;
            *(V*)&la[r * kAttPitch<T, DP> + d] = a[j];
            *(V*)&lb[r * kAttPitch<T, DP> + d] = b[j];
        }
    }
};

// over the lanes that hold the same column
template <class A, class T> __device__ __forceinline__ T across_max(T x) {
    if constexpr (A::M == 16) {
        const T y = __shfl_xor(x, 16);
        x = y > x ? y : x;
    }
    const T y = __shfl_xor(x, 32);
    return y > x ? y : x;
}
template <class A, class T> __device__ __forceinline__ T across_sum(T x) {
    if constexpr (A::M == 16) x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// address of row r (of the G Lq rows of key head hk)
template <class T>
__device__ __forceinline__ int64_t att_row(const AttArgs<T>& p, const Strides4& s, int b, int hk, uint32_t r) {
    uint32_t g = 0, i = r;
    if (p.G > 1) {
        g = r / (uint32_t)p.Lq;
        i = r - g * (uint32_t)p.Lq;
    }
    return b * s.b + (int64_t)(hk * p.G + (int)g) * s.h + (int64_t)i * s.l;
}

// ---- the softmax of one tile ----------------------------------------------------------------------------------------------------------
// s: scores S^T of NS sub-tiles, becomes probabilities relative to the running maximum m; l is this lane's share of the sum.  Returns the
// factor by which what was summed before has to shrink.
template <class A, int NS>
__device__ __forceinline__ typename A::T att_softmax(typename A::Acc (&s)[NS], uint32_t word, int h, typename A::T scale_base, typename A::T& m, typename A::T& l) {
    using T = typename A::T;
    T top = -(T)__builtin_inf();
#pragma unroll
    for (int u = 0; u < NS; u++) s[u] *= scale_base;
    if (word != ~0u) {
#pragma unroll
        for (int u = 0; u < NS; u++)
#pragma unroll
            for (int r = 0; r < A::R; r++)
                if (!((word >> (u * A::M + A::acc_row(r, h))) & 1u)) s[u][r] = -(T)__builtin_inf();
    }
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
        for (int r = 0; r < A::R; r++) top = s[u][r] > top ? s[u][r] : top;
    top = across_max<A>(top);
    const T m_new = top > m ? top : m;
    const T mu = m_new == -(T)__builtin_inf() ? T(0) : m_new;   // (nothing attended to yet: every exponential below is 0)
    const T alpha = A::exp_(m - mu);
    T sum = 0;
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
        for (int r = 0; r < A::R; r++) {
            s[u][r] = A::exp_(s[u][r] - mu);
            sum += s[u][r];
        }
    l = l * alpha + sum;
    m = m_new;
    return alpha;
}

template <class A> __device__ __forceinline__ typename A::T att_lse_of(typename A::T m, typename A::T l) {
    using T = typename A::T;
    return l == T(0) ? -(T)__builtin_inf() : (T)((m + A::log_(l)) * (T)(1.0 / A::kBase));
}

// Stores a wavefront's result out^T (lane: row, registers: width) or its share of it; d_of(i, r) is the element that register r of
// accumulator i holds.
template <class A, int ND, class DOf>
__device__ __forceinline__ void att_store(const AttArgs<typename A::T>& p, const typename A::Acc (&o)[ND], DOf d_of, uint32_t head, int b, int hk, uint32_t row,
                                          uint32_t split, int h, typename A::T m, typename A::T l) {
    using T = typename A::T;
    if (p.splits == 1) {
        const T inv = l == T(0) ? T(0) : T(1) / l;   // a row that attends to nothing is zero
        T* orow = p.o + att_row(p, p.so, b, hk, row);
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int r = 0; r < A::R; r++)
                if (d_of(i, r) < p.Dv) orow[d_of(i, r) * p.so.d] = o[i][r] * inv;
        if (p.lse_out && h == 0) p.lse_out[att_row(p, p.slse, b, hk, row)] = att_lse_of<A>(m, l);
        return;
    }
    const size_t at = ((size_t)head * p.rows + row) * p.splits + split;
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < A::R; r++)
            if (d_of(i, r) < p.Dv) p.part_o[at * p.Dv + d_of(i, r)] = o[i][r];
    if (h == 0) {
        p.part_m[at] = m;
        p.part_l[at] = l;
    }
}

// ---- forward ------------------------------------------------------------------------------------------------------------------------------
// A wavefront owns M rows and keeps their queries in registers; the workgroup's wavefronts share the keys and values, which go through
// two LDS buffers: the next tile's loads are in flight while this one is worked on, and one barrier per tile suffices (a wavefront
// that writes buffer b has passed the barrier behind everybody's last reads of it).
template <class A, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DP <= 64 ? 2 : 1) void attention_kernel(AttArgs<typename A::T> p) {
    using T = typename A::T;
    using V = typename Vec16<T>::type;
    using Acc = typename A::Acc;
    constexpr int M = A::M, N = A::N, GN = A::G * N, NT = DP / GN, NS = kAttTile / M, ND = DP / M, P = kAttPitch<T, DP>;
    __shared__ __attribute__((aligned(16))) T Ks[2][kAttTile * P];
    __shared__ __attribute__((aligned(16))) T Vs[2][kAttTile * P];
    __shared__ uint32_t words[kAttWords];
    uint32_t head, inner;
    att_place(blockIdx.x, p.blocks * p.splits, p.B * p.Hk, &head, &inner);
    const uint32_t block = inner / p.splits, split = inner - block * p.splits;
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (M - 1), h = lane / M;
    const uint32_t row = (block * WAVES + wave) * M + c;
    const bool live = row < p.rows;
    const T* qr = p.q + att_row(p, p.sq, b, hk, live ? row : 0);
    V q[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) q[t] = att_load<T>(qr, GN * t + h * N, p.Dk, p.sq.d, p.vec);
    Acc o[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) o[i] = 0;
    T m = -(T)__builtin_inf(), l = 0;
    const int tiles = (p.Lk + kAttTile - 1) / kAttTile;
    const int t0 = split * p.split_tiles, t1 = tiles < (int)(t0 + p.split_tiles) ? tiles : (int)(t0 + p.split_tiles);
    const T* kb = p.k + b * p.sk.b + hk * p.sk.h;
    const T* vb = p.v + b * p.sv.b + hk * p.sv.h;
    AttStage<T, DP, WAVES> st;
    for (int w0 = t0; w0 < t1; w0 += kAttWords) {
        const int wn = t1 - w0 < kAttWords ? t1 - w0 : kAttWords;
        __syncthreads();
        att_words(p, b, w0, wn, words, 64 * WAVES);
        __syncthreads();
        auto next = [&](int i) {   // the next tile that has a key, from i on
            while (i < wn && __builtin_amdgcn_readfirstlane(words[i]) == 0) i++;
            return i;
        };
        auto fetch = [&](int i) {
            const int key0 = (w0 + i) * kAttTile;
            st.load([&](int r, int which) {
                const int key = key0 + r < p.Lk ? key0 + r : p.Lk - 1;
                return which ? vb + key * p.sv.l : kb + key * p.sk.l;
            }, p.Dk, p.Dv, p.sk.d, p.sv.d, p.vec, __builtin_amdgcn_readfirstlane(words[i]));
        };
        int i = next(0), buf = 0;
        if (i < wn) fetch(i);
        while (i < wn) {
            st.store(Ks[buf], Vs[buf]);
            __syncthreads();
            const uint32_t word = __builtin_amdgcn_readfirstlane(words[i]);
            i = next(i + 1);
            if (i < wn) fetch(i);
            const T *ks = Ks[buf], *vs = Vs[buf];
            Acc s[NS];
#pragma unroll
            for (int u = 0; u < NS; u++) {
                s[u] = 0;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const V a = *(const V*)&ks[(u * M + c) * P + GN * t + h * N];
#pragma unroll
                    for (int e = 0; e < N; e++) s[u] = A::mfma(a[e], q[t][e], s[u]);
                }
            }
            const T alpha = att_softmax<A, NS>(s, word, h, p.scale_base, m, l);
            if (__any(alpha != T(1))) {
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= alpha;
            }
#pragma unroll
            for (int u = 0; u < NS; u++)
#pragma unroll
                for (int r = 0; r < A::R; r++)
#pragma unroll
                    for (int d = 0; d < ND; d++) o[d] = A::mfma(vs[(u * M + A::acc_row(r, h)) * P + d * M + c], s[u][r], o[d]);
            buf ^= 1;
        }
    }
    l = across_sum<A>(l);
    if (live) att_store<A, ND>(p, o, [&](int i, int r) { return i * M + A::acc_row(r, h); }, head, b, hk, row, split, h, m, l);
}

// Few rows (a decoding step): one wavefront takes 16 rows and a share of the keys, straight from memory into the operands' registers.
// Bound by the bytes of the keys and values: 32 keys at width 64 are 2048 cycles of the matrix pipe and 16 KB, i.e. the pipes keep up with
// three times the memory's rate.  A lane of value row `key` loads elements 16-byte-wise and uses element e of load g for
// accumulator E g + e: accumulator i holds the elements E 16 g + E row + e of the result.
template <class A, int DP>
__global__ __launch_bounds__(64) void attention_few_kernel(AttArgs<typename A::T> p) {
    using T = typename A::T;
    using V = typename Vec16<T>::type;
    using Acc = typename A::Acc;
    // (double precision at width 128: 16 keys a step, 32 do not fit the registers)
    constexpr int M = A::M, N = A::N, GN = A::G * N, NT = DP / GN, NS = sizeof(T) * DP > 512 ? 1 : 2, ND = DP / M, NG = ND / N, KEYS = NS * M;
    static_assert(M == 16 && NG * N == ND, "whole loads");
    uint32_t head, inner;
    att_place(blockIdx.x, p.blocks * p.splits, p.B * p.Hk, &head, &inner);
    const uint32_t block = inner / p.splits, split = inner - block * p.splits;
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const int lane = threadIdx.x, c = lane & (M - 1), h = lane / M;
    const uint32_t row = block * M + c;
    const bool live = row < p.rows;
    const T* qr = p.q + att_row(p, p.sq, b, hk, live ? row : 0);
    V q[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) q[t] = att_load<T>(qr, GN * t + h * N, p.Dk, p.sq.d, p.vec);
    Acc o[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) o[i] = 0;
    T m = -(T)__builtin_inf(), l = 0;
    const int tiles = (p.Lk + kAttTile - 1) / kAttTile;
    const int t0 = split * p.split_tiles, t1 = tiles < (int)(t0 + p.split_tiles) ? tiles : (int)(t0 + p.split_tiles);
    const T* kb = p.k + b * p.sk.b + hk * p.sk.h;
    const T* vb = p.v + b * p.sv.b + hk * p.sv.h;
    const bool whole = p.vec && p.Dk == DP && p.Dv == DP;
    uint32_t word = t0 < t1 ? (uint32_t)__ballot(att_key_on(p, b, t0 * kAttTile + (lane & 31))) : 0u;
    for (int t = t0; t < t1; t++) {
        const uint32_t now = word;
        const bool ahead = t + 1 < t1 && att_key_on(p, b, (t + 1) * kAttTile + (lane & 31));   // the next tile's word, read beside this tile
#pragma unroll
        for (int part = 0; part < kAttTile / KEYS; part++) {
            const uint32_t on = KEYS == kAttTile ? now : (now >> (part * KEYS)) & ((1u << (KEYS & 31)) - 1u);
            if (on == 0) continue;
            const int key0 = t * kAttTile + part * KEYS;
            V ka[NS][NT], va[NS][A::R][NG];
            auto rows_of = [&](auto load) {
#pragma unroll
                for (int u = 0; u < NS; u++) {
                    const int key = key0 + u * M + c;
                    const T* kr = kb + (key < p.Lk ? key : p.Lk - 1) * p.sk.l;
#pragma unroll
                    for (int i = 0; i < NT; i++) ka[u][i] = load(kr, GN * i + h * N, p.Dk, p.sk.d);
                }
#pragma unroll
                for (int u = 0; u < NS; u++)
#pragma unroll
                    for (int r = 0; r < A::R; r++) {
                        const int key = key0 + u * M + A::acc_row(r, h);
                        const T* vr = vb + (key < p.Lk ? key : p.Lk - 1) * p.sv.l;
#pragma unroll
                        for (int g = 0; g < NG; g++) va[u][r][g] = load(vr, (16 * g + c) * N, p.Dv, p.sv.d);
                    }
            };
            if (whole) rows_of([](const T* base, int d, int, int64_t) { return *(const V*)(base + d); });
            else rows_of([&](const T* base, int d, int D, int64_t sd) { return att_load<T>(base, d, D, sd, p.vec); });
            Acc s[NS];
#pragma unroll
            for (int u = 0; u < NS; u++) {
                s[u] = 0;
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int e = 0; e < N; e++) s[u] = A::mfma(ka[u][i][e], q[i][e], s[u]);
            }
            const uint32_t mine = KEYS == kAttTile ? on : on | ~0u << (KEYS & 31);   // a full step is ~0
            const T alpha = att_softmax<A, NS>(s, mine, h, p.scale_base, m, l);
#pragma unroll
            for (int i = 0; i < ND; i++) o[i] *= alpha;
            if (mine != ~0u) {
#pragma unroll
                for (int u = 0; u < NS; u++)
#pragma unroll
                    for (int r = 0; r < A::R; r++)
                        if (!((on >> (u * M + A::acc_row(r, h))) & 1u)) {
#pragma unroll
                            for (int g = 0; g < NG; g++) va[u][r][g] = 0;
                        }
            }
#pragma unroll
            for (int u = 0; u < NS; u++)
#pragma unroll
                for (int r = 0; r < A::R; r++)
#pragma unroll
                    for (int i = 0; i < ND; i++) o[i] = A::mfma(va[u][r][i / N][i % N], s[u][r], o[i]);
        }
        word = (uint32_t)__ballot(ahead);
    }
    l = across_sum<A>(l);
    if (live) att_store<A, ND>(p, o, [&](int i, int r) { return 16 * N * (i / N) + N * A::acc_row(r, h) + i % N; }, head, b, hk, row, split, h, m, l);
}

// Joins the shares of each row: a wavefront per row, first the shares' weights across its lanes, then lanes along the width.
template <class A>
__global__ __launch_bounds__(256) void attention_join_kernel(AttArgs<typename A::T> p) {
    using T = typename A::T;
    __shared__ T weights[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t row = (size_t)blockIdx.x * 4 + wave;
    if (row >= (size_t)p.B * p.Hk * p.rows) return;   // (no barrier below: a wavefront uses its own weights only)
    const uint32_t head = (uint32_t)(row / p.rows), r = (uint32_t)(row - (size_t)head * p.rows);
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const bool in = (uint32_t)lane < p.splits;         // at most 64 shares
    const T pm = in ? p.part_m[row * p.splits + lane] : -(T)__builtin_inf(), pl = in ? p.part_l[row * p.splits + lane] : T(0);
    T m = pm;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T y = __shfl_xor(m, d);
        m = y > m ? y : m;
    }
    const T w = A::exp_(pm - (m == -(T)__builtin_inf() ? T(0) : m));
    T l = w * pl;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
    weights[wave][lane] = l == T(0) ? T(0) : w / l;
    __builtin_amdgcn_wave_barrier();
    T* orow = p.o + att_row(p, p.so, b, hk, r);
    const T* part = p.part_o + row * p.splits * p.Dv;
    for (int d = lane; d < p.Dv; d += 64) {
        T o = 0;
#pragma unroll 8
        for (uint32_t s = 0; s < p.splits; s++) o += weights[wave][s] * part[(size_t)s * p.Dv + d];
        orow[d * p.so.d] = o;
    }
    if (p.lse_out && lane == 0) p.lse_out[att_row(p, p.slse, b, hk, r)] = att_lse_of<A>(m, l);
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------------
// delta[row] = sum_d d_out out, 16 lanes a row
template <class T>
__global__ __launch_bounds__(256) void attention_delta_kernel(AttArgs<T> p) {
    const size_t row = (size_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int lane = threadIdx.x & 15;
    const bool live = row < (size_t)p.B * p.Hk * p.rows;
    double sum = 0;
    if (live) {
        const uint32_t head = (uint32_t)(row / p.rows), r = (uint32_t)(row - (size_t)head * p.rows);
        const int b = head / p.Hk, hk = head - b * p.Hk;
        const T *x = p.out + att_row(p, p.so, b, hk, r), *y = p.d_out + att_row(p, p.sdo, b, hk, r);
        for (int d = lane; d < p.Dv; d += 16) sum += (double)x[d * p.so.d] * (double)y[d * p.sdo.d];
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor(sum, d);
    if (live && lane == 0) p.delta[row] = (T)sum;
}

// The exponent's base-scaled lse of a row; +inf for a row that attends to nothing, so that its probabilities are 0.
template <class A> __device__ __forceinline__ typename A::T att_lse(typename A::T lse) {
    using T = typename A::T;
    return lse == -(T)__builtin_inf() ? (T)__builtin_inf() : (T)(lse * (T)A::kBase);
}

constexpr int kGradWaves = 4;
template <class T, int DP> struct GradLds {
    T a[2][kAttTile * kAttPitch<T, DP>];
    T b[2][kAttTile * kAttPitch<T, DP>];
    T lse[2][kAttTile], delta[2][kAttTile];
    uint32_t words[kAttWords];
};

// dq: a wavefront owns M rows and walks the keys, as the forward pass does.
template <class A, int DP>
__device__ __forceinline__ void att_dq(const AttArgs<typename A::T>& p, GradLds<typename A::T, DP>& lds, uint32_t at) {
    using T = typename A::T;
    using V = typename Vec16<T>::type;
    using Acc = typename A::Acc;
    constexpr int M = A::M, N = A::N, GN = A::G * N, NT = DP / GN, NS = kAttTile / M, ND = DP / M, P = kAttPitch<T, DP>, WAVES = kGradWaves;
    uint32_t head, inner;
    att_place(at, p.blocks * p.splits, p.B * p.Hk, &head, &inner);
    const uint32_t block = inner / p.splits, split = inner - block * p.splits;
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (M - 1), h = lane / M;
    const uint32_t row = (block * WAVES + wave) * M + c;
    const bool live = row < p.rows;
    V q[NT], g[NT];
    const T* qr = p.q + att_row(p, p.sq, b, hk, live ? row : 0);
    const T* gr = p.d_out + att_row(p, p.sdo, b, hk, live ? row : 0);
#pragma unroll
    for (int t = 0; t < NT; t++) {
        q[t] = att_load<T>(qr, GN * t + h * N, p.Dk, p.sq.d, p.vec);
        g[t] = att_load<T>(gr, GN * t + h * N, p.Dv, p.sdo.d, p.vec);
    }
    const T lse = live ? att_lse<A>(p.lse[att_row(p, p.slse, b, hk, row)]) : (T)__builtin_inf();
    const T delta = live ? p.delta[(size_t)head * p.rows + row] : T(0);
    Acc dq[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) dq[i] = 0;
    const int tiles = (p.Lk + kAttTile - 1) / kAttTile;
    const int t0 = split * p.split_tiles, t1 = tiles < (int)(t0 + p.split_tiles) ? tiles : (int)(t0 + p.split_tiles);
    const T* kb = p.k + b * p.sk.b + hk * p.sk.h;
    const T* vb = p.v + b * p.sv.b + hk * p.sv.h;
    AttStage<T, DP, WAVES> st;
    for (int w0 = t0; w0 < t1; w0 += kAttWords) {
        const int wn = t1 - w0 < kAttWords ? t1 - w0 : kAttWords;
        __syncthreads();
        att_words(p, b, w0, wn, lds.words, 64 * WAVES);
        __syncthreads();
        auto next = [&](int i) {
            while (i < wn && __builtin_amdgcn_readfirstlane(lds.words[i]) == 0) i++;
            return i;
        };
        auto fetch = [&](int i) {
            const int key0 = (w0 + i) * kAttTile;
            st.load([&](int r, int which) {
                const int key = key0 + r < p.Lk ? key0 + r : p.Lk - 1;
                return which ? vb + key * p.sv.l : kb + key * p.sk.l;
            }, p.Dk, p.Dv, p.sk.d, p.sv.d, p.vec, __builtin_amdgcn_readfirstlane(lds.words[i]));
        };
        int i = next(0), buf = 0;
        if (i < wn) fetch(i);
        while (i < wn) {
            st.store(lds.a[buf], lds.b[buf]);
            __syncthreads();
            const uint32_t word = __builtin_amdgcn_readfirstlane(lds.words[i]);
            i = next(i + 1);
            if (i < wn) fetch(i);
            const T *ks = lds.a[buf], *vs = lds.b[buf];
#pragma unroll
            for (int u = 0; u < NS; u++) {
                Acc s = 0, dp = 0;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const V a = *(const V*)&ks[(u * M + c) * P + GN * t + h * N];
                    const V w = *(const V*)&vs[(u * M + c) * P + GN * t + h * N];
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        s = A::mfma(a[e], q[t][e], s);
                        dp = A::mfma(w[e], g[t][e], dp);
                    }
                }
#pragma unroll
                for (int r = 0; r < A::R; r++) s[r] = A::exp_(s[r] * p.scale_base - lse) * (dp[r] - delta) * p.scale;
                if (word != ~0u) {
#pragma unroll
                    for (int r = 0; r < A::R; r++)
                        if (!((word >> (u * M + A::acc_row(r, h))) & 1u)) s[r] = 0;
                }
#pragma unroll
                for (int r = 0; r < A::R; r++)
#pragma unroll
                    for (int d = 0; d < ND; d++) dq[d] = A::mfma(ks[(u * M + A::acc_row(r, h)) * P + d * M + c], s[r], dq[d]);
            }
            buf ^= 1;
        }
    }
    if (!live) return;
    T* o;
    int64_t sd;
    if (p.splits == 1) {
        o = p.dq + att_row(p, p.sdq, b, hk, row);
        sd = p.sdq.d;
    } else {
        o = p.part_dq + (((size_t)split * p.B * p.Hk + head) * p.rows + row) * p.Dk;
        sd = 1;
    }
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < A::R; r++) {
            const int d = i * M + A::acc_row(r, h);
            if (d < p.Dk) o[d * sd] = dq[i][r];
        }
}

// dk and dv: a wavefront owns M keys and walks the rows of the group's query heads.
template <class A, int DP>
__device__ __forceinline__ void att_dkv(const AttArgs<typename A::T>& p, GradLds<typename A::T, DP>& lds, uint32_t at) {
    using T = typename A::T;
    using V = typename Vec16<T>::type;
    using Acc = typename A::Acc;
    constexpr int M = A::M, N = A::N, GN = A::G * N, NT = DP / GN, NS = kAttTile / M, ND = DP / M, P = kAttPitch<T, DP>, WAVES = kGradWaves;
    uint32_t head, inner;
    att_place(at, p.kblocks * p.ksplits, p.B * p.Hk, &head, &inner);
    const uint32_t block = inner / p.ksplits, split = inner - block * p.ksplits;
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (M - 1), h = lane / M;
    const int key = (block * WAVES + wave) * M + c;
    const bool in = key < p.Lk, on = att_key_on(p, b, key);
    V k[NT], v[NT];
    {
        const T* kr = p.k + b * p.sk.b + hk * p.sk.h + (in ? key : 0) * p.sk.l;
        const T* vr = p.v + b * p.sv.b + hk * p.sv.h + (in ? key : 0) * p.sv.l;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            k[t] = att_load<T>(kr, GN * t + h * N, p.Dk, p.sk.d, p.vec);
            v[t] = att_load<T>(vr, GN * t + h * N, p.Dv, p.sv.d, p.vec);
            if (!on) k[t] = v[t] = 0;
        }
    }
    Acc dk[ND], dv[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) dk[i] = dv[i] = 0;
    const int tiles = ((int)p.rows + kAttTile - 1) / kAttTile;
    const int t0 = split * p.ksplit_tiles, t1 = tiles < (int)(t0 + p.ksplit_tiles) ? tiles : (int)(t0 + p.ksplit_tiles);
    const bool any = __syncthreads_or((int)on);   // a block whose keys are all masked has nothing to add up
    AttStage<T, DP, WAVES> st;
    T lse = 0, delta = 0;                          // of row threadIdx.x of the tile in flight
    auto fetch = [&](int t) {
        const uint32_t r0 = (uint32_t)t * kAttTile, left = p.rows - r0;
        st.load([&](int r, int which) {
            const uint32_t at_row = r0 + r < p.rows ? r0 + r : p.rows - 1;
            return which ? p.d_out + att_row(p, p.sdo, b, hk, at_row) : p.q + att_row(p, p.sq, b, hk, at_row);
        }, p.Dk, p.Dv, p.sq.d, p.sdo.d, p.vec, left >= 32 ? ~0u : (1u << left) - 1u);
        if (threadIdx.x < kAttTile) {
            const uint32_t r = r0 + threadIdx.x;
            lse = r < p.rows ? att_lse<A>(p.lse[att_row(p, p.slse, b, hk, r)]) : (T)__builtin_inf();
            delta = r < p.rows ? p.delta[(size_t)head * p.rows + r] : T(0);
        }
    };
    int buf = 0;
    if (any && t0 < t1) fetch(t0);
    for (int t = t0; any && t < t1; t++) {
        st.store(lds.a[buf], lds.b[buf]);
        if (threadIdx.x < kAttTile) {
            lds.lse[buf][threadIdx.x] = lse;
            lds.delta[buf][threadIdx.x] = delta;
        }
        __syncthreads();
        if (t + 1 < t1) fetch(t + 1);
        const T *qs = lds.a[buf], *gs = lds.b[buf];
#pragma unroll
        for (int u = 0; u < NS; u++) {
            Acc s = 0, dp = 0;
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const V a = *(const V*)&qs[(u * M + c) * P + GN * i + h * N];
                const V w = *(const V*)&gs[(u * M + c) * P + GN * i + h * N];
#pragma unroll
                for (int e = 0; e < N; e++) {
                    s = A::mfma(a[e], k[i][e], s);
                    dp = A::mfma(w[e], v[i][e], dp);
                }
            }
#pragma unroll
            for (int r = 0; r < A::R; r++) {
                const int i = u * M + A::acc_row(r, h);
                const T pr = on ? A::exp_(s[r] * p.scale_base - lds.lse[buf][i]) : T(0);
                dp[r] = on ? pr * (dp[r] - lds.delta[buf][i]) * p.scale : T(0);
                s[r] = pr;
            }
#pragma unroll
            for (int r = 0; r < A::R; r++)
#pragma unroll
                for (int i = 0; i < ND; i++) {
                    const int at_lds = (u * M + A::acc_row(r, h)) * P + i * M + c;
                    dv[i] = A::mfma(gs[at_lds], s[r], dv[i]);
                    dk[i] = A::mfma(qs[at_lds], dp[r], dk[i]);
                }
        }
        buf ^= 1;
    }
    if (!in) return;
    T *ok, *ov;
    int64_t sk, sv;
    if (p.ksplits == 1) {
        ok = p.dk + b * p.sdk.b + hk * p.sdk.h + (int64_t)key * p.sdk.l;
        ov = p.dv + b * p.sdv.b + hk * p.sdv.h + (int64_t)key * p.sdv.l;
        sk = p.sdk.d;
        sv = p.sdv.d;
    } else {
        const size_t at_row = ((size_t)split * p.B * p.Hk + head) * p.Lk + key;
        ok = p.part_dk + at_row * p.Dk;
        ov = p.part_dv + at_row * p.Dv;
        sk = sv = 1;
    }
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < A::R; r++) {
            const int d = i * M + A::acc_row(r, h);
            if (d < p.Dk) ok[d * sk] = dk[i][r];
            if (d < p.Dv) ov[d * sv] = dv[i][r];
        }
}

// Both halves of the backward pass in one launch: the workgroups of dk and dv first (they are the longer ones), then those of dq, so that
// neither half leaves compute units idle while the other runs out.
template <class A, int DP>
__global__ __launch_bounds__(64 * kGradWaves, DP <= 64 ? 2 : 1) void attention_grad_kernel(AttArgs<typename A::T> p, uint32_t kv_workgroups) {
    __shared__ __attribute__((aligned(16))) GradLds<typename A::T, DP> lds;
    if (blockIdx.x < kv_workgroups) att_dkv<A, DP>(p, lds, blockIdx.x);
    else att_dq<A, DP>(p, lds, blockIdx.x - kv_workgroups);
}

// Adds up the shares: workgroups [0, kv) take rows of dk and dv, the others rows of dq; a thread per element.
template <class T>
__global__ __launch_bounds__(256) void attention_grad_join_kernel(AttArgs<T> p, uint32_t kv_workgroups) {
    const bool kv = blockIdx.x < kv_workgroups;
    const size_t i = ((size_t)blockIdx.x - (kv ? 0 : kv_workgroups)) * 256 + threadIdx.x;
    const uint32_t len = kv ? (uint32_t)p.Lk : p.rows, width = (uint32_t)(kv ? p.Dk + p.Dv : p.Dk), shares = kv ? p.ksplits : p.splits;
    const size_t heads = (size_t)p.B * p.Hk, row = i / width;
    if (row >= heads * len) return;
    uint32_t d = (uint32_t)(i - row * width);
    const bool second = kv && d >= (uint32_t)p.Dk;
    if (second) d -= p.Dk;
    const uint32_t w = second ? p.Dv : p.Dk;
    const T* part = (second ? p.part_dv : kv ? p.part_dk : p.part_dq) + row * w + d;
    T sum = 0;
#pragma unroll 4
    for (uint32_t s = 0; s < shares; s++) sum += part[(size_t)s * heads * len * w];
    const uint32_t head = (uint32_t)(row / len), r = (uint32_t)(row - (size_t)head * len);
    const int b = head / p.Hk, hk = head - b * p.Hk;
    if (!kv) p.dq[att_row(p, p.sdq, b, hk, r) + d * p.sdq.d] = sum;
    else if (second) p.dv[b * p.sdv.b + hk * p.sdv.h + (int64_t)r * p.sdv.l + d * p.sdv.d] = sum;
    else p.dk[b * p.sdk.b + hk * p.sdk.h + (int64_t)r * p.sdk.l + d * p.sdk.d] = sum;
}

// ---- plan and launch ------------------------------------------------------------------------------------------------------------------------
constexpr uint32_t kAttCUs = 256;   // MI355X; a constant, so that the size of the scratch memory can be asked for without a device
constexpr int64_t kFewRows = 32;    // up to here the kernel without LDS (two blocks of 16 rows read the keys twice, the second time from the L2)

// Shares of a walk over `tiles` tiles, at least two tiles each and at most `most` shares, until `want` workgroups are reached.
inline void att_shares(int64_t workgroups, int64_t tiles, int64_t want, int64_t most, uint32_t* shares, uint32_t* share_tiles) {
    int64_t n = workgroups >= want || workgroups < 1 ? 1 : (want + workgroups - 1) / workgroups;
    if (n > (tiles + 1) / 2) n = (tiles + 1) / 2;
    if (n > most) n = most;
    if (n < 1) n = 1;
    int64_t each = (tiles + n - 1) / n;
    if (each < 1) each = 1;
    n = (tiles + each - 1) / each;
    *shares = (uint32_t)(n < 1 ? 1 : n);
    *share_tiles = (uint32_t)each;
}

struct AttPlan {
    int waves;   // 0: the kernel for few rows
    uint32_t blocks, splits, split_tiles;
    size_t o_bytes, m_bytes, total;
};
template <class T> AttPlan att_plan(int64_t heads, int64_t rows, int64_t Lk, int64_t Dv) {
    constexpr int M = MmaOf<T>::Tile::M;
    AttPlan p;
    const int64_t tiles = (Lk + kAttTile - 1) / kAttTile;
    if (rows <= kFewRows) {
        p.waves = 0;
        p.blocks = cdiv(rows, 16);
        att_shares(heads * p.blocks, tiles, 8 * kAttCUs, 64, &p.splits, &p.split_tiles);    // two wavefronts per SIMD
    } else {
        p.waves = rows <= 2 * M ? 2 : 4;
        p.blocks = cdiv(rows, (int64_t)p.waves * M);
        att_shares(heads * p.blocks, tiles, 2 * kAttCUs * 4 / p.waves / 2, 64, &p.splits, &p.split_tiles);
    }
    const size_t parts = (size_t)heads * rows * p.splits;
    p.o_bytes = up256(parts * Dv * sizeof(T));
    p.m_bytes = up256(parts * sizeof(T));
    p.total = p.splits > 1 ? p.o_bytes + 2 * p.m_bytes : 0;
    return p;
}

struct AttGradPlan {
    uint32_t blocks, splits, split_tiles, kblocks, ksplits, ksplit_tiles;
    size_t delta_bytes, dq_bytes, dk_bytes, dv_bytes, total;
};
template <class T> AttGradPlan att_grad_plan(int64_t heads, int64_t rows, int64_t Lk, int64_t Dk, int64_t Dv) {
    constexpr int M = MmaOf<T>::Tile::M;
    AttGradPlan p;
    p.blocks = cdiv(rows, kGradWaves * M);
    p.kblocks = cdiv(Lk, kGradWaves * M);
    att_shares(heads * p.blocks, (Lk + kAttTile - 1) / kAttTile, kAttCUs, 64, &p.splits, &p.split_tiles);
    att_shares(heads * p.kblocks, (rows + kAttTile - 1) / kAttTile, kAttCUs, 64, &p.ksplits, &p.ksplit_tiles);
    p.delta_bytes = up256((size_t)heads * rows * sizeof(T));
    p.dq_bytes = p.splits > 1 ? up256((size_t)p.splits * heads * rows * Dk * sizeof(T)) : 0;
    p.dk_bytes = p.ksplits > 1 ? up256((size_t)p.ksplits * heads * Lk * Dk * sizeof(T)) : 0;
    p.dv_bytes = p.ksplits > 1 ? up256((size_t)p.ksplits * heads * Lk * Dv * sizeof(T)) : 0;
    p.total = p.delta_bytes + p.dq_bytes + p.dk_bytes + p.dv_bytes;
    return p;
}

template <class T> int32_t attention_forward(AttArgs<T>& p, void* scratch, size_t scratch_bytes, hipStream_t s);
template <class T> int32_t attention_backward(AttArgs<T>& p, void* scratch, size_t scratch_bytes, hipStream_t s);

// fn(std::integral_constant<int, DP>) for the padded width: instantiated widths are multiples of the tile edge
template <class T, class Fn> void att_widths(int width, Fn fn) {
    if (sizeof(T) == 8 && width <= 16) fn(std::integral_constant<int, sizeof(T) == 8 ? 16 : 32>());
    else if (width <= 32) fn(std::integral_constant<int, 32>());
    else if (sizeof(T) == 8 && width <= 48) fn(std::integral_constant<int, sizeof(T) == 8 ? 48 : 64>());
    else if (width <= 64) fn(std::integral_constant<int, 64>());
    else if (width <= 96) fn(std::integral_constant<int, 96>());
    else fn(std::integral_constant<int, 128>());
}

template <class T> int32_t attention_forward_impl(AttArgs<T>& p, void* scratch, size_t scratch_bytes, hipStream_t s) {
    using Tile = typename MmaOf<T>::Tile;
    using Few = typename MmaOf<T>::Few;
    const uint32_t heads = (uint32_t)(p.B * p.Hk);
    const AttPlan pl = att_plan<T>(heads, p.rows, p.Lk, p.Dv);
    p.blocks = pl.blocks;
    p.splits = pl.splits;
    p.split_tiles = pl.split_tiles;
    char* ws = nullptr;
    WorkspaceLease lease;
    DNH_TRY(get_scratch(s, pl.total, scratch, scratch_bytes, (void**)&ws, lease, "dnh_cross_attention"));
    p.part_o = (T*)ws;
    p.part_m = (T*)(ws + pl.o_bytes);
    p.part_l = (T*)(ws + pl.o_bytes + pl.m_bytes);
    const dim3 grid(heads * p.blocks * p.splits);
    const int width = p.Dk > p.Dv ? p.Dk : p.Dv;
    if (pl.waves == 0) {
        if (width <= 64) hipLaunchKernelGGL((attention_few_kernel<Few, 64>), grid, dim3(64), 0, s, p);
        else hipLaunchKernelGGL((attention_few_kernel<Few, 128>), grid, dim3(64), 0, s, p);
    } else {
        att_widths<T>(width, [&](auto dp) {
            if (pl.waves == 2) hipLaunchKernelGGL((attention_kernel<Tile, dp.value, 2>), grid, dim3(128), 0, s, p);
            else hipLaunchKernelGGL((attention_kernel<Tile, dp.value, 4>), grid, dim3(256), 0, s, p);
        });
    }
    DNH_LAUNCH_CHECK();
    if (p.splits > 1) {
        hipLaunchKernelGGL((attention_join_kernel<Tile>), dim3(cdiv((int64_t)heads * p.rows, 4)), dim3(256), 0, s, p);
        DNH_LAUNCH_CHECK();
    }
    return DNH_OK;
}

template <class T> int32_t attention_backward_impl(AttArgs<T>& p, void* scratch, size_t scratch_bytes, hipStream_t s) {
    using Tile = typename MmaOf<T>::Tile;
    const int64_t heads = (int64_t)p.B * p.Hk;
    const AttGradPlan pl = att_grad_plan<T>(heads, p.rows, p.Lk, p.Dk, p.Dv);
    p.blocks = pl.blocks;
    p.splits = pl.splits;
    p.split_tiles = pl.split_tiles;
    p.kblocks = pl.kblocks;
    p.ksplits = pl.ksplits;
    p.ksplit_tiles = pl.ksplit_tiles;
    char* ws = nullptr;
    WorkspaceLease lease;
    DNH_TRY(get_scratch(s, pl.total, scratch, scratch_bytes, (void**)&ws, lease, "dnh_cross_attention_grad"));
    p.delta = (T*)ws;
    p.part_dq = (T*)(ws + pl.delta_bytes);
    p.part_dk = (T*)(ws + pl.delta_bytes + pl.dq_bytes);
    p.part_dv = (T*)(ws + pl.delta_bytes + pl.dq_bytes + pl.dk_bytes);
    if (p.rows) {
        hipLaunchKernelGGL((attention_delta_kernel<T>), dim3(cdiv(heads * p.rows, 16)), dim3(256), 0, s, p);
        DNH_LAUNCH_CHECK();
    }
    const uint32_t kv = p.dk ? (uint32_t)heads * p.kblocks * p.ksplits : 0, dq = p.dq ? (uint32_t)heads * p.blocks * p.splits : 0;
    if (kv + dq == 0) return DNH_OK;
    att_widths<T>(p.Dk > p.Dv ? p.Dk : p.Dv, [&](auto dp) {
        hipLaunchKernelGGL((attention_grad_kernel<Tile, dp.value>), dim3(kv + dq), dim3(64 * kGradWaves), 0, s, p, kv);
    });
    DNH_LAUNCH_CHECK();
    const unsigned jkv = p.dk && p.ksplits > 1 ? cdiv(heads * p.Lk * (p.Dk + p.Dv), 256) : 0, jdq = p.dq && p.splits > 1 ? cdiv(heads * p.rows * p.Dk, 256) : 0;
    if (jkv + jdq) {
        hipLaunchKernelGGL((attention_grad_join_kernel<T>), dim3(jkv + jdq), dim3(256), 0, s, p, jkv);
        DNH_LAUNCH_CHECK();
    }
    return DNH_OK;
}

template <> int32_t attention_forward<float>(AttArgs<float>&, void*, size_t, hipStream_t);
template <> int32_t attention_backward<float>(AttArgs<float>&, void*, size_t, hipStream_t);
template <> int32_t attention_forward<double>(AttArgs<double>&, void*, size_t, hipStream_t);
template <> int32_t attention_backward<double>(AttArgs<double>&, void*, size_t, hipStream_t);

}  // namespace dnh
