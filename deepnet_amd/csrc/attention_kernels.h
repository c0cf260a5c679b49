// Cross attention on the matrix cores: kernels and their launcher for one element type (attention.hip: single precision and the entry
// points, attention_f64.hip: double precision).
//
// Queries [B; Hq; Lq; Dk], keys [B; Hk; Lk; Dk], values [B; Hk; Lk; Dv], Hq = G Hk: the G query heads of a key head form one list of
// G Lq rows, so keys and values are staged once for all of them and their gradients are summed over the group by construction.
//
//   S = scale q k^T     P = softmax over the keys that the mask [B; Lk] leaves     out = P v     lse = log sum e^S
//   delta = sum_d d_out out    dS = scale P (d_out v^T - delta)    dq = dS k    dk = dS^T q    dv = P^T d_out
//
// Matrix instructions v_mfma_f32_32x32x2_f32 / v_mfma_f64_16x16x4_f64: lane l supplies A[l % M][l / M] and B[l / M][l % M] and holds
// column l % M of the result, in register r the row acc_row(r, l / M).  The products are arranged so that nothing is transposed:
// a wavefront computes S^T (keys down, queries across), so the maximum and the sum of a query are over a lane's own registers and
// its M-distant neighbours, and register r of P^T is, as it stands, the B operand of the step of out^T = v^T P^T that runs over the keys
// { acc_row(r, 0), acc_row(r, 1), ... }.  The backward kernels use the same property with queries and keys in either role.
#pragma once

#include "model_ops.h"

namespace dnh {

template <class T> struct Mma;
template <> struct Mma<float> {
    static constexpr int M = 32, G = 2, R = 16, N = 4;   // tile edge, lane groups (= K of the instruction), registers, elements of 16 bytes
    typedef float Acc __attribute__((ext_vector_type(16)));
    static __device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }
    static __device__ __forceinline__ Acc mfma(float a, float b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
    // exponentials in base 2: the logarithm's base goes into the scale
    static __device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x); }
    static __device__ __forceinline__ float log_(float x) { return __log2f(x); }
    static constexpr double kBase = 1.44269504088896340736;   // log of e in that base
};
template <> struct Mma<double> {
    static constexpr int M = 16, G = 4, R = 4, N = 2;
    typedef double Acc __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ int acc_row(int r, int h) { return 4 * r + h; }
    static __device__ __forceinline__ Acc mfma(double a, double b, Acc c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ double exp_(double x) { return exp(x); }
    static __device__ __forceinline__ double log_(double x) { return log(x); }
    static constexpr double kBase = 1.0;
};

constexpr int kAttTile = 32;   // keys (forward, dq) or query rows (dk, dv) of one step
constexpr int kAttMaxWaves = 4;

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
    uint32_t blocks;          // row blocks (forward, dq) or key blocks (dk, dv) of one key head
    uint32_t splits, split_tiles;   // forward: workgroups that share a row block's keys, and the tiles of each
    T *part_o, *part_m, *part_l;    // their results
    T* delta;
};

// Which (batch, key head) and which block of it a workgroup takes: workgroups go to the eight XCDs in turn, and each XCD gets a
// contiguous range, so the blocks that read the same keys and values share an L2.
__device__ __forceinline__ bool att_place(uint32_t per, uint32_t heads, uint32_t* head, uint32_t* inner) {
    const uint32_t total = per * heads, each = (total + 7) / 8;
    const uint32_t at = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= each || at >= total) return false;
    *head = at / per;
    *inner = at - *head * per;
    return true;
}
inline unsigned att_grid(uint32_t per, uint32_t heads) { return 8 * ((per * heads + 7) / 8); }

// 16 bytes of a row at element d, zeros beyond D
template <class T>
__device__ __forceinline__ typename Vec16<T>::type att_load(const T* row, int d, int D, int64_t sd, bool vec) {
    using V = typename Vec16<T>::type;
    constexpr int N = Mma<T>::N;
    if (vec && d + N <= D) return *(const V*)(row + d);
    V v = 0;
#pragma unroll
    for (int e = 0; e < N; e++)
        if (d + e < D) v[e] = row[(int64_t)(d + e) * sd];
    return v;
}

template <class T, int DP> constexpr int kAttPitch = DP + Mma<T>::N;   // LDS rows: 16 rows' 16-byte reads fall on different banks

// The 32-bit word of which of a tile's keys are attended to
template <class T>
__device__ __forceinline__ uint32_t att_keys(const AttArgs<T>& p, int b, int key0) {
    const int lane = threadIdx.x & 63, key = key0 + (lane & 31);
    bool ok = key < p.Lk;
    if (ok && p.mask) ok = p.mask[b * p.mask_b + key * p.mask_l] != 0;
    return (uint32_t)__ballot(ok);
}

// rows [0, 32) of a tile into LDS; rows whose bit is not set become zeros (and are not read)
template <class T, int DP>
__device__ __forceinline__ void att_stage(T* lds, const T* base, int64_t sl, int64_t sd, int D, bool vec, uint32_t word) {
    using V = typename Vec16<T>::type;
    constexpr int N = Mma<T>::N, PER = DP / N;
    for (int i = threadIdx.x; i < kAttTile * PER; i += blockDim.x) {
        const int r = i / PER, d = (i - r * PER) * N;
        V v = 0;
        if ((word >> r) & 1u) v = att_load<T>(base + (int64_t)r * sl, d, D, sd, vec);
        *(V*)&lds[r * kAttPitch<T, DP> + d] = v;
    }
}

template <class T> __device__ __forceinline__ T across(T x, bool maximum) {   // over the lanes that hold the same column
    if constexpr (Mma<T>::M == 16) {
        const T y = __shfl_xor(x, 16);
        x = maximum ? (y > x ? y : x) : x + y;
    }
    const T y = __shfl_xor(x, 32);
    return maximum ? (y > x ? y : x) : x + y;
}

// address of row r (of the G Lq rows of key head hk)
template <class T>
__device__ __forceinline__ int64_t att_row(const AttArgs<T>& p, const Strides4& s, int b, int hk, uint32_t r) {
    const uint32_t g = r / (uint32_t)p.Lq, i = r - g * (uint32_t)p.Lq;
    return b * s.b + (int64_t)(hk * p.G + (int)g) * s.h + (int64_t)i * s.l;
}

// ---- forward ------------------------------------------------------------------------------------------------------------------------------
// A wavefront owns M rows; the workgroup's wavefronts share the staged keys and values.
template <class T, int DP>
__global__ __launch_bounds__(64 * kAttMaxWaves) void attention_kernel(AttArgs<T> p) {
    using A = Mma<T>;
    using V = typename Vec16<T>::type;
    using Acc = typename A::Acc;
    constexpr int M = A::M, N = A::N, NT = DP / 8, NS = kAttTile / M, ND = DP / M;
    __shared__ __attribute__((aligned(16))) T Ks[kAttTile][kAttPitch<T, DP>];
    __shared__ __attribute__((aligned(16))) T Vs[kAttTile][kAttPitch<T, DP>];
    uint32_t head, inner;
    if (!att_place(p.blocks * p.splits, p.B * p.Hk, &head, &inner)) return;
    const uint32_t block = inner / p.splits, split = inner - block * p.splits;
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (M - 1), h = lane / M;
    const uint32_t row = (block * (blockDim.x >> 6) + wave) * M + c;
    const bool live = row < p.rows;
    V q[NT];
    {
        const T* qr = p.q + (live ? att_row(p, p.sq, b, hk, row) : 0);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            q[t] = 0;
            if (live) q[t] = att_load<T>(qr, 8 * t + h * N, p.Dk, p.sq.d, p.vec);
        }
    }
    Acc o[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) o[i] = 0;
    T m = -(T)__builtin_inf(), l = 0;
    const int tiles = (p.Lk + kAttTile - 1) / kAttTile;
    const int t0 = split * p.split_tiles, t1 = tiles < (int)(t0 + p.split_tiles) ? tiles : (int)(t0 + p.split_tiles);
    const T* kb = p.k + b * p.sk.b + hk * p.sk.h;
    const T* vb = p.v + b * p.sv.b + hk * p.sv.h;
    for (int t = t0; t < t1; t++) {
        const int key0 = t * kAttTile;
        const uint32_t word = att_keys(p, b, key0);
        if (word == 0) continue;   // the same for the whole workgroup
        __syncthreads();
        att_stage<T, DP>(&Ks[0][0], kb + (int64_t)key0 * p.sk.l, p.sk.l, p.sk.d, p.Dk, p.vec, word);
        att_stage<T, DP>(&Vs[0][0], vb + (int64_t)key0 * p.sv.l, p.sv.l, p.sv.d, p.Dv, p.vec, word);
        __syncthreads();
        Acc s[NS];
#pragma unroll
        for (int u = 0; u < NS; u++) {
            s[u] = 0;
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const V a = *(const V*)&Ks[u * M + c][8 * i + h * N];
#pragma unroll
                for (int e = 0; e < N; e++) s[u] = A::mfma(a[e], q[i][e], s[u]);
            }
        }
        T top = -(T)__builtin_inf();
#pragma unroll
        for (int u = 0; u < NS; u++)
#pragma unroll
            for (int r = 0; r < A::R; r++) {
                T x = s[u][r] * p.scale_base;
                if (!((word >> (u * M + A::acc_row(r, h))) & 1u)) x = -(T)__builtin_inf();
                s[u][r] = x;
                top = x > top ? x : top;
            }
        top = across(top, true);
        const T m_new = top > m ? top : m;
        const T mu = m_new == -(T)__builtin_inf() ? T(0) : m_new;
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
        if (__any(alpha != T(1))) {
#pragma unroll
            for (int i = 0; i < ND; i++) o[i] *= alpha;
        }
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int u = 0; u < NS; u++)
#pragma unroll
                for (int r = 0; r < A::R; r++) o[i] = A::mfma(Vs[u * M + A::acc_row(r, h)][i * M + c], s[u][r], o[i]);
    }
    l = across(l, false);
    if (!live) return;
    if (p.splits == 1) {
        const T inv = l == T(0) ? T(0) : T(1) / l;   // a row that attends to nothing is zero
        T* orow = p.o + att_row(p, p.so, b, hk, row);
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int r = 0; r < A::R; r++) {
                const int d = i * M + A::acc_row(r, h);
                if (d < p.Dv) orow[d * p.so.d] = o[i][r] * inv;
            }
        if (p.lse_out && h == 0)
            p.lse_out[att_row(p, p.slse, b, hk, row)] = l == T(0) ? -(T)__builtin_inf() : (T)((m + A::log_(l)) * (T)(1.0 / A::kBase));
        return;
    }
    const size_t at = ((size_t)head * p.rows + row) * p.splits + split;
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < A::R; r++) {
            const int d = i * M + A::acc_row(r, h);
            if (d < p.Dv) p.part_o[at * p.Dv + d] = o[i][r];
        }
    if (h == 0) {
        p.part_m[at] = m;
        p.part_l[at] = l;
    }
}

// Joins the splits of each row: 64 threads, a row each wavefront, lanes along the width.
template <class T>
__global__ __launch_bounds__(256) void attention_join_kernel(AttArgs<T> p) {
    using A = Mma<T>;
    const int lane = threadIdx.x & 63;
    const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (size_t)p.B * p.Hk * p.rows) return;
    const uint32_t head = (uint32_t)(row / p.rows), r = (uint32_t)(row - (size_t)head * p.rows);
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const T *pm = p.part_m + row * p.splits, *pl = p.part_l + row * p.splits;
    T m = -(T)__builtin_inf();
    for (uint32_t s = 0; s < p.splits; s++) m = pm[s] > m ? pm[s] : m;
    const T mu = m == -(T)__builtin_inf() ? T(0) : m;
    T l = 0;
    for (uint32_t s = 0; s < p.splits; s++) l += A::exp_(pm[s] - mu) * pl[s];
    const T inv = l == T(0) ? T(0) : T(1) / l;
    T* orow = p.o + att_row(p, p.so, b, hk, r);
    for (int d = lane; d < p.Dv; d += 64) {
        T o = 0;
        for (uint32_t s = 0; s < p.splits; s++) o += A::exp_(pm[s] - mu) * p.part_o[(row * p.splits + s) * p.Dv + d];
        orow[d * p.so.d] = o * inv;
    }
    if (p.lse_out && lane == 0) p.lse_out[att_row(p, p.slse, b, hk, r)] = l == T(0) ? -(T)__builtin_inf() : (T)((m + A::log_(l)) * (T)(1.0 / A::kBase));
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
template <class T> __device__ __forceinline__ T att_lse(T lse) {
    return lse == -(T)__builtin_inf() ? (T)__builtin_inf() : (T)(lse * (T)Mma<T>::kBase);
}

// dq: a wavefront owns M rows and walks the keys, as the forward pass does.
template <class T, int DP>
__global__ __launch_bounds__(64 * kAttMaxWaves) void attention_dq_kernel(AttArgs<T> p) {
    using A = Mma<T>;
    using V = typename Vec16<T>::type;
    using Acc = typename A::Acc;
    constexpr int M = A::M, N = A::N, NT = DP / 8, NS = kAttTile / M, ND = DP / M;
    __shared__ __attribute__((aligned(16))) T Ks[kAttTile][kAttPitch<T, DP>];
    __shared__ __attribute__((aligned(16))) T Vs[kAttTile][kAttPitch<T, DP>];
    uint32_t head, block;
    if (!att_place(p.blocks, p.B * p.Hk, &head, &block)) return;
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (M - 1), h = lane / M;
    const uint32_t row = (block * (blockDim.x >> 6) + wave) * M + c;
    const bool live = row < p.rows;
    V q[NT], g[NT];
    T lse = (T)__builtin_inf(), delta = 0;
    {
        const T* qr = p.q + (live ? att_row(p, p.sq, b, hk, row) : 0);
        const T* gr = p.d_out + (live ? att_row(p, p.sdo, b, hk, row) : 0);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            q[t] = 0;
            g[t] = 0;
            if (live) {
                q[t] = att_load<T>(qr, 8 * t + h * N, p.Dk, p.sq.d, p.vec);
                g[t] = att_load<T>(gr, 8 * t + h * N, p.Dv, p.sdo.d, p.vec);
            }
        }
        if (live) {
            lse = att_lse(p.lse[att_row(p, p.slse, b, hk, row)]);
            delta = p.delta[(size_t)head * p.rows + row];
        }
    }
    Acc dq[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) dq[i] = 0;
    const int tiles = (p.Lk + kAttTile - 1) / kAttTile;
    const T* kb = p.k + b * p.sk.b + hk * p.sk.h;
    const T* vb = p.v + b * p.sv.b + hk * p.sv.h;
    for (int t = 0; t < tiles; t++) {
        const int key0 = t * kAttTile;
        const uint32_t word = att_keys(p, b, key0);
        if (word == 0) continue;
        __syncthreads();
        att_stage<T, DP>(&Ks[0][0], kb + (int64_t)key0 * p.sk.l, p.sk.l, p.sk.d, p.Dk, p.vec, word);
        att_stage<T, DP>(&Vs[0][0], vb + (int64_t)key0 * p.sv.l, p.sv.l, p.sv.d, p.Dv, p.vec, word);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NS; u++) {
            Acc s = 0, dp = 0;
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const V a = *(const V*)&Ks[u * M + c][8 * i + h * N];
                const V w = *(const V*)&Vs[u * M + c][8 * i + h * N];
#pragma unroll
                for (int e = 0; e < N; e++) {
                    s = A::mfma(a[e], q[i][e], s);
                    dp = A::mfma(w[e], g[i][e], dp);
                }
            }
#pragma unroll
            for (int r = 0; r < A::R; r++) {
                const T pr = A::exp_(s[r] * p.scale_base - lse);
                const bool on = (word >> (u * M + A::acc_row(r, h))) & 1u;
                s[r] = on ? pr * (dp[r] - delta) * p.scale : T(0);
            }
#pragma unroll
            for (int i = 0; i < ND; i++)
#pragma unroll
                for (int r = 0; r < A::R; r++) dq[i] = A::mfma(Ks[u * M + A::acc_row(r, h)][i * M + c], s[r], dq[i]);
        }
    }
    if (!live) return;
    T* o = p.dq + att_row(p, p.sdq, b, hk, row);
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < A::R; r++) {
            const int d = i * M + A::acc_row(r, h);
            if (d < p.Dk) o[d * p.sdq.d] = dq[i][r];
        }
}

// dk and dv: a wavefront owns M keys and walks the rows of the group's query heads.
template <class T, int DP>
__global__ __launch_bounds__(64 * kAttMaxWaves) void attention_dkv_kernel(AttArgs<T> p) {
    using A = Mma<T>;
    using V = typename Vec16<T>::type;
    using Acc = typename A::Acc;
    constexpr int M = A::M, N = A::N, NT = DP / 8, NS = kAttTile / M, ND = DP / M;
    __shared__ __attribute__((aligned(16))) T Qs[kAttTile][kAttPitch<T, DP>];
    __shared__ __attribute__((aligned(16))) T Gs[kAttTile][kAttPitch<T, DP>];
    __shared__ T lse_s[kAttTile], delta_s[kAttTile];
    uint32_t head, block;
    if (!att_place(p.blocks, p.B * p.Hk, &head, &block)) return;
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (M - 1), h = lane / M;
    const int key = (block * (blockDim.x >> 6) + wave) * M + c;
    const bool in = key < p.Lk, on = in && (!p.mask || p.mask[b * p.mask_b + key * p.mask_l] != 0);
    V k[NT], v[NT];
    {
        const T* kr = p.k + b * p.sk.b + hk * p.sk.h + (int64_t)(on ? key : 0) * p.sk.l;
        const T* vr = p.v + b * p.sv.b + hk * p.sv.h + (int64_t)(on ? key : 0) * p.sv.l;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            k[t] = 0;
            v[t] = 0;
            if (on) {
                k[t] = att_load<T>(kr, 8 * t + h * N, p.Dk, p.sk.d, p.vec);
                v[t] = att_load<T>(vr, 8 * t + h * N, p.Dv, p.sv.d, p.vec);
            }
        }
    }
    Acc dk[ND], dv[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) dk[i] = dv[i] = 0;
    const bool any = __syncthreads_or((int)on);   // a block whose keys are all masked has nothing to add up
    for (uint32_t r0 = 0; any && r0 < p.rows; r0 += kAttTile) {
        __syncthreads();
        for (int i = threadIdx.x; i < kAttTile * (DP / N); i += blockDim.x) {
            const int r = i / (DP / N), d = (i - r * (DP / N)) * N;
            V x = 0, y = 0;
            if (r0 + r < p.rows) {
                x = att_load<T>(p.q + att_row(p, p.sq, b, hk, r0 + r), d, p.Dk, p.sq.d, p.vec);
                y = att_load<T>(p.d_out + att_row(p, p.sdo, b, hk, r0 + r), d, p.Dv, p.sdo.d, p.vec);
            }
            *(V*)&Qs[r][d] = x;
            *(V*)&Gs[r][d] = y;
        }
        if (threadIdx.x < kAttTile) {
            const uint32_t r = r0 + threadIdx.x;
            lse_s[threadIdx.x] = r < p.rows ? att_lse(p.lse[att_row(p, p.slse, b, hk, r)]) : (T)__builtin_inf();
            delta_s[threadIdx.x] = r < p.rows ? p.delta[(size_t)head * p.rows + r] : T(0);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NS; u++) {
            Acc s = 0, dp = 0;
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const V a = *(const V*)&Qs[u * M + c][8 * i + h * N];
                const V w = *(const V*)&Gs[u * M + c][8 * i + h * N];
#pragma unroll
                for (int e = 0; e < N; e++) {
                    s = A::mfma(a[e], k[i][e], s);
                    dp = A::mfma(w[e], v[i][e], dp);
                }
            }
#pragma unroll
            for (int r = 0; r < A::R; r++) {
                const int i = u * M + A::acc_row(r, h);
                const T pr = on ? A::exp_(s[r] * p.scale_base - lse_s[i]) : T(0);
                dp[r] = on ? pr * (dp[r] - delta_s[i]) * p.scale : T(0);
                s[r] = pr;
            }
#pragma unroll
            for (int i = 0; i < ND; i++)
#pragma unroll
                for (int r = 0; r < A::R; r++) {
                    dv[i] = A::mfma(Gs[u * M + A::acc_row(r, h)][i * M + c], s[r], dv[i]);
                    dk[i] = A::mfma(Qs[u * M + A::acc_row(r, h)][i * M + c], dp[r], dk[i]);
                }
        }
    }
    if (!in) return;
    T* ok = p.dk + b * p.sdk.b + hk * p.sdk.h + (int64_t)key * p.sdk.l;
    T* ov = p.dv + b * p.sdv.b + hk * p.sdv.h + (int64_t)key * p.sdv.l;
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < A::R; r++) {
            const int d = i * M + A::acc_row(r, h);
            if (d < p.Dk) ok[d * p.sdk.d] = dk[i][r];
            if (d < p.Dv) ov[d * p.sdv.d] = dv[i][r];
        }
}

// ---- plan and launch ------------------------------------------------------------------------------------------------------------------------
// Wavefronts of a workgroup: as many as the rows (or keys) of a head fill, up to four.
inline int att_waves(int64_t n, int M) {
    const int64_t w = (n + M - 1) / M;
    return w >= 4 ? 4 : w >= 2 ? 2 : 1;
}
constexpr uint32_t kAttCUs = 256;   // MI355X; a constant, so that the size of the scratch memory can be asked for without a device

struct AttPlan {
    int waves;
    uint32_t blocks, splits, split_tiles;
    size_t o_bytes, m_bytes, total;
};
template <class T> AttPlan att_plan(int64_t heads, int64_t rows, int64_t Lk, int64_t Dv) {
    AttPlan p;
    p.waves = att_waves(rows, Mma<T>::M);
    p.blocks = cdiv(rows, (int64_t)p.waves * Mma<T>::M);
    const int64_t tiles = (Lk + kAttTile - 1) / kAttTile, wgs = heads * p.blocks;
    // keys are shared out when the row blocks do not give every SIMD two wavefronts; a share is at least two tiles
    const int64_t want = 8 * kAttCUs / p.waves;
    int64_t splits = wgs >= want / 2 ? 1 : (want + wgs - 1) / wgs;
    const int64_t most = (tiles + 1) / 2;
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    p.split_tiles = (uint32_t)((tiles + splits - 1) / splits);
    if (p.split_tiles < 1) p.split_tiles = 1;
    p.splits = (uint32_t)((tiles + p.split_tiles - 1) / p.split_tiles);
    if (p.splits < 1) p.splits = 1;
    const size_t parts = (size_t)heads * rows * p.splits;
    p.o_bytes = up256(parts * Dv * sizeof(T));
    p.m_bytes = up256(parts * sizeof(T));
    p.total = p.splits > 1 ? p.o_bytes + 2 * p.m_bytes : 0;
    return p;
}

template <class T> int32_t attention_forward(AttArgs<T>& p, void* scratch, size_t scratch_bytes, hipStream_t s);
template <class T> int32_t attention_backward(AttArgs<T>& p, void* scratch, size_t scratch_bytes, hipStream_t s);

template <class T, int DP> void launch_forward(const AttArgs<T>& p, int waves, hipStream_t s) {
    hipLaunchKernelGGL((attention_kernel<T, DP>), dim3(att_grid(p.blocks * p.splits, p.B * p.Hk)), dim3(64 * waves), 0, s, p);
}
template <class T, int DP> void launch_dq(const AttArgs<T>& p, int waves, hipStream_t s) {
    hipLaunchKernelGGL((attention_dq_kernel<T, DP>), dim3(att_grid(p.blocks, p.B * p.Hk)), dim3(64 * waves), 0, s, p);
}
template <class T, int DP> void launch_dkv(const AttArgs<T>& p, int waves, hipStream_t s) {
    hipLaunchKernelGGL((attention_dkv_kernel<T, DP>), dim3(att_grid(p.blocks, p.B * p.Hk)), dim3(64 * waves), 0, s, p);
}
// instantiations by padded width: multiples of the tile edge
#define DNH_ATT_DISPATCH(T, FN, p, waves, s)                                     \
    do {                                                                         \
        const int _w = (p).Dk > (p).Dv ? (p).Dk : (p).Dv;                        \
        if (sizeof(T) == 8 && _w <= 16) FN<T, sizeof(T) == 8 ? 16 : 32>(p, waves, s);      \
        else if (_w <= 32) FN<T, 32>(p, waves, s);                               \
        else if (sizeof(T) == 8 && _w <= 48) FN<T, sizeof(T) == 8 ? 48 : 64>(p, waves, s); \
        else if (_w <= 64) FN<T, 64>(p, waves, s);                               \
        else if (_w <= 96) FN<T, 96>(p, waves, s);                               \
        else FN<T, 128>(p, waves, s);                                            \
    } while (0)

template <class T> int32_t attention_forward_impl(AttArgs<T>& p, void* scratch, size_t scratch_bytes, hipStream_t s) {
    const AttPlan pl = att_plan<T>((int64_t)p.B * p.Hk, p.rows, p.Lk, p.Dv);
    p.blocks = pl.blocks;
    p.splits = pl.splits;
    p.split_tiles = pl.split_tiles;
    char* ws = nullptr;
    WorkspaceLease lease;
    DNH_TRY(get_scratch(s, pl.total, scratch, scratch_bytes, (void**)&ws, lease, "dnh_cross_attention"));
    p.part_o = (T*)ws;
    p.part_m = (T*)(ws + pl.o_bytes);
    p.part_l = (T*)(ws + pl.o_bytes + pl.m_bytes);
    DNH_ATT_DISPATCH(T, launch_forward, p, pl.waves, s);
    DNH_LAUNCH_CHECK();
    if (p.splits > 1) {
        hipLaunchKernelGGL((attention_join_kernel<T>), dim3(cdiv((int64_t)p.B * p.Hk * p.rows, 4)), dim3(256), 0, s, p);
        DNH_LAUNCH_CHECK();
    }
    return DNH_OK;
}

template <class T> int32_t attention_backward_impl(AttArgs<T>& p, void* scratch, size_t scratch_bytes, hipStream_t s) {
    const int64_t heads = (int64_t)p.B * p.Hk;
    WorkspaceLease lease;
    DNH_TRY(get_scratch(s, up256((size_t)heads * p.rows * sizeof(T)), scratch, scratch_bytes, (void**)&p.delta, lease, "dnh_cross_attention_grad"));
    if (p.rows) {
        hipLaunchKernelGGL((attention_delta_kernel<T>), dim3(cdiv(heads * p.rows, 16)), dim3(256), 0, s, p);
        DNH_LAUNCH_CHECK();
    }
    if (p.dq && p.rows) {
        const int waves = att_waves(p.rows, Mma<T>::M);
        p.blocks = cdiv(p.rows, waves * Mma<T>::M);
        DNH_ATT_DISPATCH(T, launch_dq, p, waves, s);
        DNH_LAUNCH_CHECK();
    }
    if (p.dk && p.Lk) {
        const int waves = att_waves(p.Lk, Mma<T>::M);
        p.blocks = cdiv(p.Lk, waves * Mma<T>::M);
        DNH_ATT_DISPATCH(T, launch_dkv, p, waves, s);
        DNH_LAUNCH_CHECK();
    }
    return DNH_OK;
}

template <> int32_t attention_forward<float>(AttArgs<float>&, void*, size_t, hipStream_t);
template <> int32_t attention_backward<float>(AttArgs<float>&, void*, size_t, hipStream_t);
template <> int32_t attention_forward<double>(AttArgs<double>&, void*, size_t, hipStream_t);
template <> int32_t attention_backward<double>(AttArgs<double>&, void*, size_t, hipStream_t);

}  // namespace dnh
