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
    uint32_t lq_mul;          // r / Lq = r lq_mul >> lq_shift for r < 2^31
    int lq_shift;
    T scale, scale_base;      // scale, and scale x log e in the exponentials' base
    bool vec;                 // q, k, v (and d_out) are contiguous along their last axis
    bool whole;               // and their widths are whole 16-byte pieces
    bool exact;               // no bf16 parts
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

// The same without a branch (which would make every load wait for the one before it), for rows that are contiguous and hold whole pieces
template <class T, bool WHOLE>
__device__ __forceinline__ typename Vec16<T>::type att_piece(const T* row, int d, int D, int64_t sd, bool vec) {
    using V = typename Vec16<T>::type;
    if constexpr (WHOLE) {
        const V v = *(const V*)(row + (d < D ? d : 0));
        return d < D ? v : V(0);
    } else {
        return att_load<T>(row, d, D, sd, vec);
    }
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

// A tile of 32 rows of two matrices on its way from memory to LDS: loaded into registers while the tile before it is worked on.  WHOLE:
// rows are contiguous and hold whole 16-byte pieces; the loads are then straight-line code whose results nothing touches before
// store() (a branch between two ways of loading would make the compiler wait for the data where the ways meet).
template <class T, int DP, int WAVES, bool WHOLE> struct AttStage {
    using V = typename Vec16<T>::type;
    static constexpr int N = kVecN<T>, PER = DP / N, NL = kAttTile * PER / (64 * WAVES);
    static_assert(NL * 64 * WAVES == kAttTile * PER, "the workgroup covers a tile evenly");
    V a[NL], b[NL];
    // row(r, which): address of row r of the tile (always readable)
    template <class Row> __device__ __forceinline__ void load(Row row, int Da, int Db, int64_t sda, int64_t sdb, bool vec) {
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const int i = threadIdx.x + j * 64 * WAVES, r = i / PER, d = (i - r * PER) * N;
            const T *pa = row(r, 0), *pb = row(r, 1);
            if constexpr (WHOLE) {
                a[j] = *(const V*)(pa + (d < Da ? d : 0));
                b[j] = *(const V*)(pb + (d < Db ? d : 0));
            } else {
                a[j] = att_load<T>(pa, d, Da, sda, vec);
                b[j] = att_load<T>(pb, d, Db, sdb, vec);
            }
        }
    }
    // row and first element of the thread's piece j
    __device__ __forceinline__ int row_of(int j) const { return (threadIdx.x + j * 64 * WAVES) / PER; }
    __device__ __forceinline__ int elem_of(int j) const { return (threadIdx.x + j * 64 * WAVES - row_of(j) * PER) * N; }
    // rows whose bit is not set, and what lies beyond the width, become zeros
    __device__ __forceinline__ void clear_off(int Da, int Db, uint32_t word) {
        if (word != ~0u || Da < DP || Db < DP) {
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const bool on = (word >> row_of(j)) & 1u;
                if (!on || elem_of(j) >= Da) a[j] = 0;
                if (!on || elem_of(j) >= Db) b[j] = 0;
            }
        }
    }
    __device__ __forceinline__ void store(T* la, T* lb, int Da, int Db, uint32_t word) {
        clear_off(Da, Db, word);
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const int at = row_of(j) * kAttPitch<T, DP> + elem_of(j);
            *(V*)&la[at] = a[j];
            *(V*)&lb[at] = b[j];
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
        g = (uint32_t)(((uint64_t)r * p.lq_mul) >> p.lq_shift);   // r / Lq
        i = r - g * (uint32_t)p.Lq;
    }
    return b * s.b + (int64_t)(hk * p.G + (int)g) * s.h + (int64_t)i * s.l;
}

// ---- products of one staged tile ------------------------------------------------------------------------------------------------------
// The compiler, left alone, reads an operand from LDS right before the instructions that use it and waits; with one or two wavefronts on
// a SIMD the matrix pipe then idles for the LDS latency each time.  Here every read is issued one or two groups of instructions
// ahead, and scheduling barriers (which let ordinary vector and scalar instructions pass) keep it there.
//
// Result accumulators: lane row i of accumulator n holds element d_of(n, i) of the width, chosen so that a lane's operands for E
// accumulators are neighbours in LDS (one read) and its results are neighbours in memory.
template <class A, int DP, int WAVES = 4, bool WHOLE = true> struct AttOps {
    using Mma = A;
    using T = typename A::T;
    using V = typename Vec16<T>::type;
    using Acc = typename A::Acc;
    static constexpr int M = A::M, N = A::N, GN = A::G * N, NT = DP / GN, NS = kAttTile / M, ND = DP / M, P = kAttPitch<T, DP>;
    struct Watch {};                                   // (nothing that these instructions could not multiply)
    static __device__ __forceinline__ bool failed(const Watch&) { return false; }
    struct __attribute__((aligned(16))) Tile {
        T x[kAttTile * P];
    };
    struct Operand {                                   // a row of the other matrix: element [t][e] is GN t + h N + e
        V v[NT];
    };
    static __device__ __forceinline__ void load(Operand& q, const T* row, int D, int64_t sd, bool vec, int h, Watch&) {
#pragma unroll
        for (int t = 0; t < NT; t++) q.v[t] = att_piece<T, WHOLE>(row, GN * t + h * N, D, sd, vec);
    }
    static __device__ __forceinline__ void clear(Operand& q) {
#pragma unroll
        for (int t = 0; t < NT; t++) q.v[t] = 0;
    }
    using Stage = AttStage<T, DP, WAVES, WHOLE>;
    static __device__ __forceinline__ void store(Stage& st, Tile& a, Tile& b, int Da, int Db, uint32_t word, Watch&) { st.store(a.x, b.x, Da, Db, word); }
    static constexpr int E = ND % N == 0 ? N : ND == 2 ? 2 : 1, NE = ND / E;
    typedef T VE __attribute__((ext_vector_type(E)));
    static __device__ __forceinline__ int d_of(int n, int i) { return (n / E) * (M * E) + E * i + n % E; }
    static __device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0x6); }

    // a lane's column of the result, times f, to a row of D elements
    static __device__ __forceinline__ void put(T* row, int64_t sd, int D, const Acc (&o)[ND], T f, int h) {
        if (E > 1 && sd == 1 && D % E == 0) {
            typedef T VU __attribute__((ext_vector_type(E), aligned(sizeof(T))));   // E neighbours at the element's alignment
#pragma unroll
            for (int n = 0; n < ND; n += E)
#pragma unroll
                for (int r = 0; r < A::R; r++) {
                    const int d = d_of(n, A::acc_row(r, h));
                    VU v;
#pragma unroll
                    for (int e = 0; e < E; e++) v[e] = o[n + e][r] * f;
                    if (d < D) *(VU*)(row + d) = v;
                }
            return;
        }
#pragma unroll
        for (int n = 0; n < ND; n++)
#pragma unroll
            for (int r = 0; r < A::R; r++) {
                const int d = d_of(n, A::acc_row(r, h));
                if (d < D) row[d * sd] = o[n][r] * f;
            }
    }
    // s = rows of sub-tile u . x
    static __device__ __forceinline__ void scores(Acc& s, const Tile& tile, int u, int c, int h, const Operand& q) {
        const T* at = tile.x + (u * M + c) * P + h * N;
        const V(&x)[NT] = q.v;
        V a[2];
        a[0] = *(const V*)at;
        s = 0;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (t + 1 < NT) a[(t + 1) & 1] = *(const V*)(at + GN * (t + 1));
            pin();
#pragma unroll
            for (int e = 0; e < N; e++) s = A::mfma(a[t & 1][e], x[t][e], s);
            pin();
        }
    }
    // two at once
    static __device__ __forceinline__ void scores(Acc& s, const Tile& tile, const Operand& q, Acc& z, const Tile& ztile, const Operand& g, int u, int c, int h) {
        const T *at = tile.x + (u * M + c) * P + h * N, *zat = ztile.x + (u * M + c) * P + h * N;
        const V(&x)[NT] = q.v;
        const V(&y)[NT] = g.v;
        V a[2], w[2];
        a[0] = *(const V*)at;
        w[0] = *(const V*)zat;
        s = 0;
        z = 0;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (t + 1 < NT) {
                a[(t + 1) & 1] = *(const V*)(at + GN * (t + 1));
                w[(t + 1) & 1] = *(const V*)(zat + GN * (t + 1));
            }
            pin();
#pragma unroll
            for (int e = 0; e < N; e++) {
                s = A::mfma(a[t & 1][e], x[t][e], s);
                z = A::mfma(w[t & 1][e], y[t][e], z);
            }
            pin();
        }
    }
    // operands of step x (of NS R): the tile's row that register x % R of sub-tile x / R stands for; at: element [0][E c]
    struct Row {
        VE v[NE];
        __device__ __forceinline__ void read(const T* at, int x, int h) {
            const T* r = at + ((x / A::R) * M + A::acc_row(x % A::R, h)) * P;
#pragma unroll
            for (int n = 0; n < NE; n++) v[n] = *(const VE*)(r + n * M * E);
        }
        __device__ __forceinline__ T operator[](int n) const {
            if constexpr (E == 1) return v[n][0];
            else return v[n / E][n % E];
        }
    };
    // o += (rows of sub-tile u)^T . s
    static __device__ __forceinline__ void outer(Acc (&o)[ND], const Tile& tile, const Acc& s, int u, int c, int h) {
        const T* at = tile.x + E * c;
        const int x0 = u * A::R;
        Row a[3];
        a[0].read(at, x0, h);
        a[1].read(at, x0 + 1, h);
#pragma unroll
        for (int r = 0; r < A::R; r++) {
            if (r + 2 < A::R) a[(r + 2) % 3].read(at, x0 + r + 2, h);
            pin();
#pragma unroll
            for (int n = 0; n < ND; n++) o[n] = A::mfma(a[r % 3][n], s[r], o[n]);
            pin();
        }
    }
    // two at once
    static __device__ __forceinline__ void outer(Acc (&o)[ND], const Tile& tile, const Acc& s, Acc (&z)[ND], const Tile& ztile, const Acc& y, int u, int c, int h) {
        const T *at = tile.x + E * c, *zat = ztile.x + E * c;
        const int x0 = u * A::R;
        Row a[2], w[2];
        a[0].read(at, x0, h);
        w[0].read(zat, x0, h);
#pragma unroll
        for (int r = 0; r < A::R; r++) {
            if (r + 1 < A::R) {
                a[(r + 1) & 1].read(at, x0 + r + 1, h);
                w[(r + 1) & 1].read(zat, x0 + r + 1, h);
            }
            pin();
#pragma unroll
            for (int n = 0; n < ND; n++) {
                o[n] = A::mfma(a[r & 1][n], s[r], o[n]);
                z[n] = A::mfma(w[r & 1][n], y[r], z[n]);
            }
            pin();
        }
    }
};

// ---- the same in single precision on the bf16 matrix instructions ---------------------------------------------------------------------
// v_mfma_f32_32x32x16_bf16 does in 32 cycles what v_mfma_f32_32x32x2_f32 does in 512.  A float is the exact sum of three bf16 numbers (each
// the remainder so far, rounded to nearest: 8 + 8 + 8 significant bits), every product of two parts is exact in the instruction, and of the nine
// partial products the six largest are kept: those dropped are below 2^-23 |a b| together (2 u of one rounded product), and 6 x 32 cycles take
// the place of 512.  The last part of an element below 2^-109 falls under bf16's smallest denormal: a workgroup that meets one (zero
// apart) starts again on the float instructions.  So does one whose sums are not finite: an element that rounds to an infinity in 8 bits, and an
// infinite one, has NaN as its last part.  Probabilities, which float exponentials flush at 2^-126, are kept to 2^-134; dS is scaled (kAttUp).
//
// The instruction's K = 16: lane l supplies A[l % 32][8 (l / 32) + i] and B[8 (l / 32) + i][l % 32], i = 0 .. 7.  Its result lies as that of
// v_mfma_f32_32x32x2_f32, so registers 8 j .. 8 j + 7 of lane half h are the rows 16 j + 4 h + { 0 .. 3, 8 .. 11 }: with K numbered in this order
// they are, cut, the B operand of step j of the second product.  Its A operand is the staged tile transposed, four rows of one column a lane:
// that is what ds_read_b64_tr_b16 delivers (of 16 lanes, lane x supplies the address of row x / 4, columns 4 (x % 4) .. + 3, and gets column x
// of the four rows), so one copy of the tile serves both products.
typedef __bf16 Bf8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ void cut2(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    typedef float F2 __attribute__((ext_vector_type(2)));
    typedef __bf16 B2 __attribute__((ext_vector_type(2)));
    hi = __builtin_bit_cast(uint32_t, __builtin_convertvector((F2{x, y}), B2));
    x -= __uint_as_float(hi << 16);
    y -= __uint_as_float(hi & 0xFFFF0000u);
    mid = __builtin_bit_cast(uint32_t, __builtin_convertvector((F2{x, y}), B2));
    x -= __uint_as_float(mid << 16);
    y -= __uint_as_float(mid & 0xFFFF0000u);
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((F2{x, y}), B2));
}
template <int DP, int WAVES> struct AttOpsX3 {
    using Mma = MmaF32;
    using T = float;
    using Acc = MmaF32::Acc;
    using V = Vec16<float>::type;
    static constexpr int M = 32, NS = 1, ND = DP / 32, NT = DP / 16;
    // LDS rows of 20 or 52 words beyond a multiple of 64: 16 rows' 16-byte reads fall on different banks, and the four rows of a transposed read
    // overlap little (width 128, 4 words: 311 us forward instead of 304, 330 us of gradient instead of 328).  At width 64 two workgroups have no room for that: 36 words.
    static constexpr int P = DP == 128 ? 168 : DP + 8, PLANE = kAttTile * P;
    typedef uint32_t U2 __attribute__((ext_vector_type(2)));
    typedef uint32_t U4 __attribute__((ext_vector_type(4)));
    typedef uint16_t H2 __attribute__((ext_vector_type(2)));
    struct Watch {                                     // the least first part that is not zero: -2 times it, which loses its sign, is the largest
        H2 least = 0;
        __device__ __forceinline__ void see(uint32_t hi) {
            H2 x;
            asm("v_pk_mul_lo_u16 %0, %1, %2" : "=v"(x) : "v"(hi), "s"(0xFFFEFFFEu));   // (the compiler makes a shift and a subtraction of it)
            least = __builtin_elementwise_max(least, x);
        }
    };
    // 2^-109 (a first part that was rounded up to it comes from 2^-109 (1 - 2^-9), which has parts, too)
    static __device__ __forceinline__ bool failed(const Watch& w) { return w.least[0] > 0x10000 - 2 * 0x0900 || w.least[1] > 0x10000 - 2 * 0x0900; }
    struct __attribute__((aligned(16))) Tile {
        uint16_t x[3 * PLANE];
    };
    struct Operand {                                   // element [part][t][i] of a row is 16 t + 8 h + i
        Bf8 v[3][NT];
    };
    static __device__ __forceinline__ void cut8(const float (&x)[8], Bf8 (&y)[3], Watch* w) {
        U4 part[3];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            uint32_t hi, mid, lo;
            cut2(x[2 * e], x[2 * e + 1], hi, mid, lo);
            if (w) w->see(hi);
            part[0][e] = hi;
            part[1][e] = mid;
            part[2][e] = lo;
        }
#pragma unroll
        for (int k = 0; k < 3; k++) y[k] = __builtin_bit_cast(Bf8, part[k]);
    }
    static __device__ __forceinline__ void load(Operand& q, const float* row, int D, int64_t sd, bool vec, int h, Watch& w) {
        V f[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int k = 0; k < 2; k++) f[t][k] = att_piece<float, true>(row, 16 * t + 8 * h + 4 * k, D, sd, vec);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float x[8];
            Bf8 y[3];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = f[t][i / 4][i % 4];
            cut8(x, y, &w);
#pragma unroll
            for (int k = 0; k < 3; k++) q.v[k][t] = y[k];
        }
    }
    static __device__ __forceinline__ void clear(Operand& q) {
#pragma unroll
        for (int k = 0; k < 3; k++)
#pragma unroll
            for (int t = 0; t < NT; t++) q.v[k][t] = __builtin_bit_cast(Bf8, U4(0));
    }
    using Stage = AttStage<float, DP, WAVES, true>;
    static __device__ __forceinline__ void store(Stage& st, Tile& a, Tile& b, int Da, int Db, uint32_t word, Watch& w) {
        st.clear_off(Da, Db, word);
#pragma unroll
        for (int j = 0; j < Stage::NL; j++) {
            const int at = st.row_of(j) * P + st.elem_of(j);
            auto put3 = [&](uint16_t* t, const V& v) {
                uint32_t h0, m0, l0, h1, m1, l1;
                cut2(v[0], v[1], h0, m0, l0);
                cut2(v[2], v[3], h1, m1, l1);
                w.see(h0);
                w.see(h1);
                *(U2*)(t + at) = U2{h0, h1};
                *(U2*)(t + at + PLANE) = U2{m0, m1};
                *(U2*)(t + at + 2 * PLANE) = U2{l0, l1};
            };
            put3(a.x, st.a[j]);
            put3(b.x, st.b[j]);
        }
    }
    // Reads stay ahead of the matrix instructions (as above), which go before the other wavefront's softmax: gradient of 16 x 16 heads, 512 queries,
    // 1024 keys at width 64 580 us, 595 us as the compiler orders it; at width 32 (8 x 16 heads) 152 and 155 us.
    static __device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0x6); }
    template <int P> static __device__ __forceinline__ void hold() { __builtin_amdgcn_s_setprio(P); }
    static __device__ __forceinline__ Acc mfma(const Bf8& a, const Bf8& b, const Acc& c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    // c += a . b, the smallest products first
    static __device__ __forceinline__ void six(Acc& c, const Bf8 (&a)[3], const Bf8& b0, const Bf8& b1, const Bf8& b2) {
        c = mfma(a[2], b0, c);
        c = mfma(a[0], b2, c);
        c = mfma(a[1], b1, c);
        c = mfma(a[1], b0, c);
        c = mfma(a[0], b1, c);
        c = mfma(a[0], b0, c);
    }
    static __device__ __forceinline__ void read(Bf8 (&a)[3], const uint16_t* at) {
#pragma unroll
        for (int k = 0; k < 3; k++) a[k] = *(const Bf8*)(at + k * PLANE);
    }
    // rows at + { 0 .. 3, 8 .. 11 }
    static __device__ __forceinline__ void read_tr(Bf8 (&a)[3], const uint16_t* at) {
        typedef short S4 __attribute__((ext_vector_type(4)));
        typedef short S8 __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) S4* L4;
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const S4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L4)(at + k * PLANE)), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L4)(at + k * PLANE + 8 * P));
            a[k] = __builtin_bit_cast(Bf8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
    static __device__ __forceinline__ void scores(Acc& s, const Tile& tile, int, int c, int h, const Operand& q) {
        const uint16_t* at = tile.x + c * P + 8 * h;
        Bf8 a[2][3];
        read(a[0], at);
        s = 0;
        hold<1>();
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (t + 1 < NT) read(a[(t + 1) & 1], at + 16 * (t + 1));
            pin();
            six(s, a[t & 1], q.v[0][t], q.v[1][t], q.v[2][t]);
            pin();
        }
        hold<0>();
    }
    static __device__ __forceinline__ void scores(Acc& s, const Tile& tile, const Operand& q, Acc& z, const Tile& ztile, const Operand& g, int, int c, int h) {
        if constexpr (DP <= 64) {                      // (both at once would not fit the registers of two wavefronts a SIMD)
            scores(s, tile, 0, c, h, q);
            scores(z, ztile, 0, c, h, g);
            return;
        }
        const uint16_t *at = tile.x + c * P + 8 * h, *zat = ztile.x + c * P + 8 * h;
        Bf8 a[2][3], w[2][3];
        read(a[0], at);
        read(w[0], zat);
        s = 0;
        z = 0;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (t + 1 < NT) {
                read(a[(t + 1) & 1], at + 16 * (t + 1));
                read(w[(t + 1) & 1], zat + 16 * (t + 1));
            }
            pin();
            six(s, a[t & 1], q.v[0][t], q.v[1][t], q.v[2][t]);
            six(z, w[t & 1], g.v[0][t], g.v[1][t], g.v[2][t]);
            pin();
        }
    }
    static __device__ __forceinline__ void outer(Acc (&o)[ND], const Tile& tile, const Acc s, int, int c, int h) {
        const int x = c & 15;
        const uint16_t* at = tile.x + (4 * h + (x >> 2)) * P + (c & 16) + 4 * (x & 3);
        Bf8 a[2][3], y[3];
        read_tr(a[0], at);
#pragma unroll
        for (int k = 0; k < 2 * ND; k++) {
            hold<1>();
            const int j = k / ND, m = k + 1;
            if (k % ND == 0) {
                float e[8];
#pragma unroll
                for (int i = 0; i < 8; i++) e[i] = j ? s[8 + i] : s[i];   // (the constants keep the vector in registers)
                cut8(e, y, nullptr);
            }
            if (m < 2 * ND) read_tr(a[m & 1], at + (m / ND) * 16 * P + (m % ND) * 32);
            pin();
            six(o[k % ND], a[k & 1], y[0], y[1], y[2]);
            pin();
            if (k % ND == ND - 1) hold<0>();
        }
    }
    static __device__ __forceinline__ void outer(Acc (&o)[ND], const Tile& tile, const Acc& s, Acc (&z)[ND], const Tile& ztile, const Acc& y, int u, int c, int h) {
        outer(o, tile, s, u, c, h);
        outer(z, ztile, y, u, c, h);
    }
    // accumulator n holds elements 32 n .. 32 n + 31
    static __device__ __forceinline__ void put(float* row, int64_t sd, int D, const Acc (&o)[ND], float f, int h) {
#pragma unroll
        for (int n = 0; n < ND; n++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int d = 32 * n + MmaF32::acc_row(4 * g, h);
                if (d >= D) continue;                  // (widths are whole groups of four)
                if (sd == 1) {
                    V v;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = o[n][4 * g + e] * f;
                    *(V*)(row + d) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) row[(d + e) * sd] = o[n][4 * g + e] * f;
                }
            }
    }
};
// What a kernel runs first, and what instead if that fails: the same type where it cannot.
template <class A, int DP, int WAVES, bool WHOLE> struct AttFirst {
    typedef AttOps<A, DP, WAVES, WHOLE> Ops;
};
template <int DP, int WAVES> struct AttFirst<MmaF32, DP, WAVES, true> {
    typedef AttOpsX3<DP, WAVES> Ops;
};

// ---- the softmax of one tile ----------------------------------------------------------------------------------------------------------
// s: scores S^T of NS sub-tiles, becomes probabilities relative to the running maximum m; l is this lane's share of the sum.  Returns the
// factor by which what was summed before has to shrink.
template <class A, int NS>
__device__ __forceinline__ typename A::T att_softmax(typename A::Acc (&s)[NS], uint32_t word, int h, typename A::T scale_base, typename A::T& m, typename A::T& l) {
    using T = typename A::T;
    T top = -(T)__builtin_inf();
#pragma unroll
    for (int u = 0; u < NS; u++)
#pragma unroll
        for (int r = 0; r < A::R; r++) s[u][r] *= scale_base;
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

// whether none of a lane's sums is infinite or NaN
template <class Ops> __device__ __forceinline__ bool att_finite(const typename Ops::Acc (&o)[Ops::ND]) {
    typename Ops::T t = 0;
#pragma unroll
    for (int n = 0; n < Ops::ND; n++)
#pragma unroll
        for (int r = 0; r < Ops::Mma::R; r++) t += o[n][r] * typename Ops::T(0);
    return t == typename Ops::T(0);
}

// Stores a wavefront's result out^T (lane: row, registers: width) or its share of it.
template <class Ops>
__device__ __forceinline__ void att_store(const AttArgs<typename Ops::T>& p, const typename Ops::Acc (&o)[Ops::ND], uint32_t head, int b, int hk, uint32_t row,
                                          uint32_t split, int h, typename Ops::T m, typename Ops::T l) {
    using T = typename Ops::T;
    T *to, f;
    int64_t sd;
    if (p.splits == 1) {
        to = p.o + att_row(p, p.so, b, hk, row);
        sd = p.so.d;
        f = l == T(0) ? T(0) : T(1) / l;   // a row that attends to nothing is zero
        if (p.lse_out && h == 0) p.lse_out[att_row(p, p.slse, b, hk, row)] = att_lse_of<typename Ops::Mma>(m, l);
    } else {
        const size_t at = ((size_t)head * p.rows + row) * p.splits + split;
        to = p.part_o + at * p.Dv;
        sd = 1;
        f = T(1);
        if (h == 0) {
            p.part_m[at] = m;
            p.part_l[at] = l;
        }
    }
    Ops::put(to, sd, p.Dv, o, f, h);
}

// ---- forward ------------------------------------------------------------------------------------------------------------------------------
// A wavefront owns M rows and keeps their queries in registers; the workgroup's wavefronts share the keys and values, which go through
// two LDS buffers: the next tile's loads are in flight while this one is worked on, and one barrier per tile suffices (a wavefront
// that writes buffer b has passed the barrier behind everybody's last reads of it).
// Bound by the matrix pipes and the vector instructions that the wavefronts of a SIMD do not hide behind them (softmax, cutting P and the
// staged tiles): 8 x 16 heads, 512 queries, up to 1500 keys at width 64 take 126 us, pipes busy half the time (196 us on the float
// instructions, pipes busy 72 %).  Two wavefronts a workgroup only where four would not have rows, in single precision from 33 to 64: 40 queries
// over 60 000 keys of 2 heads 35.5 us, four wavefronts 37.4, but 33 queries over 2000 keys of 64 heads 34.0 and 31.1.  Beyond, four: 2000 queries
// of 32 heads 143 us, two wavefronts 242.
template <class Ops> struct AttLds {
    typename Ops::Tile k[2], v[2];
    uint32_t words[kAttWords];
};
// false: nothing is written, and the workgroup has to take the other instructions
template <class Ops, int WAVES>
__device__ __forceinline__ bool att_forward(const AttArgs<typename Ops::T>& p, AttLds<Ops>& lds) {
    using A = typename Ops::Mma;
    using T = typename A::T;
    using Acc = typename A::Acc;
    constexpr int M = A::M, NS = kAttTile / M, ND = Ops::ND;
    uint32_t head, inner;
    att_place(blockIdx.x, p.blocks * p.splits, p.B * p.Hk, &head, &inner);
    const uint32_t block = inner / p.splits, split = inner - block * p.splits;
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (M - 1), h = lane / M;
    const uint32_t row = (block * WAVES + wave) * M + c;
    const bool live = row < p.rows;
    typename Ops::Watch watch;
    typename Ops::Operand q;
    Ops::load(q, p.q + att_row(p, p.sq, b, hk, live ? row : 0), p.Dk, p.sq.d, p.vec, h, watch);
    Acc o[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) o[i] = 0;
    T m = -(T)__builtin_inf(), l = 0;
    const T scale_base = p.scale_base;
    const int tiles = (p.Lk + kAttTile - 1) / kAttTile;
    const int t0 = split * p.split_tiles, t1 = tiles < (int)(t0 + p.split_tiles) ? tiles : (int)(t0 + p.split_tiles);
    const T* kb = p.k + b * p.sk.b + hk * p.sk.h;
    const T* vb = p.v + b * p.sv.b + hk * p.sv.h;
    typename Ops::Stage st;
    for (int w0 = t0; w0 < t1; w0 += kAttWords) {
        const int wn = t1 - w0 < kAttWords ? t1 - w0 : kAttWords;
        __syncthreads();
        att_words(p, b, w0, wn, lds.words, 64 * WAVES);
        __syncthreads();
        auto next = [&](int i) {   // the next tile that has a key, from i on
            while (i < wn && __builtin_amdgcn_readfirstlane(lds.words[i]) == 0) i++;
            return i;
        };
        auto fetch = [&](int i) {
            const int key0 = (w0 + i) * kAttTile;
            st.load([&](int r, int which) {
                const int key = key0 + r < p.Lk ? key0 + r : p.Lk - 1;
                return which ? vb + key * p.sv.l : kb + key * p.sk.l;
            }, p.Dk, p.Dv, p.sk.d, p.sv.d, p.vec);
        };
        int i = next(0), buf = 0;
        if (i < wn) fetch(i);
        while (i < wn) {
            const uint32_t word = __builtin_amdgcn_readfirstlane(lds.words[i]);
            Ops::store(st, lds.k[buf], lds.v[buf], p.Dk, p.Dv, word, watch);
            __syncthreads();
            i = next(i + 1);
            if (i < wn) fetch(i);
            Acc s[NS];
#pragma unroll
            for (int u = 0; u < NS; u++) Ops::scores(s[u], lds.k[buf], u, c, h, q);
            const T alpha = att_softmax<A, NS>(s, word, h, scale_base, m, l);
            if (__any(alpha != T(1))) {
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= alpha;
            }
#pragma unroll
            for (int u = 0; u < NS; u++) Ops::outer(o, lds.v[buf], s[u], u, c, h);
            buf ^= 1;
        }
    }
    if (!std::is_empty<typename Ops::Watch>::value && __syncthreads_or((int)(Ops::failed(watch) || (live && !(att_finite<Ops>(o) && l * T(0) == T(0)))))) return false;
    l = across_sum<A>(l);
    if (live) att_store<Ops>(p, o, head, b, hk, row, split, h, m, l);
    return true;
}
template <class A, int DP, int WAVES, bool WHOLE>
__global__ __launch_bounds__(64 * WAVES, DP <= 64 ? 2 : 1) void attention_kernel(AttArgs<typename A::T> p) {
    using First = typename AttFirst<A, DP, WAVES, WHOLE>::Ops;
    using Exact = AttOps<A, DP, WAVES, WHOLE>;
    __shared__ union {
        AttLds<First> first;
        AttLds<Exact> exact;
    } lds;
    if constexpr (!std::is_same<First, Exact>::value)
        if (!p.exact && att_forward<First, WAVES>(p, lds.first)) return;
    att_forward<Exact, WAVES>(p, lds.exact);
}


// Few rows (a decoding step): one wavefront takes 16 rows and a share of the keys, straight from memory into the operands' registers.
// Bound by the bytes of the keys and values: 32 keys at width 64 are 2048 cycles of the matrix pipe and 16 KB, i.e. the pipes keep up with
// three times the memory's rate.  A lane of value row `key` loads elements 16-byte-wise and uses element e of load g for
// accumulator E g + e: accumulator i holds the elements E 16 g + E row + e of the result.
// 16 sequences of up to 2000 keys, 4 key heads at width 64 (47 MB): 14 to 15 us, and 4 us for joining the shares.  The float instructions
// stay here: cutting a tile that one wavefront uses once costs more than it saves.
template <class A, int DP, bool WHOLE>
__global__ __launch_bounds__(64) void attention_few_kernel(AttArgs<typename A::T> p) {
    using T = typename A::T;
    using V = typename Vec16<T>::type;
    using Acc = typename A::Acc;
    // (double precision at width 128: 16 keys a step, 32 do not fit the registers)
    constexpr int M = A::M, N = A::N, GN = A::G * N, NT = DP / GN, NS = sizeof(T) * DP > 512 ? 1 : 2, ND = DP / M, NG = ND / N, KEYS = NS * M;
    static_assert(M == 16 && NG * N == ND && AttOps<A, DP>::E == N, "whole loads");
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
    for (int t = 0; t < NT; t++) q[t] = att_piece<T, WHOLE>(qr, GN * t + h * N, p.Dk, p.sq.d, p.vec);
    Acc o[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) o[i] = 0;
    T m = -(T)__builtin_inf(), l = 0;
    const int tiles = (p.Lk + kAttTile - 1) / kAttTile;
    const int t0 = split * p.split_tiles, t1 = tiles < (int)(t0 + p.split_tiles) ? tiles : (int)(t0 + p.split_tiles);
    const T* kb = p.k + b * p.sk.b + hk * p.sk.h;
    const T* vb = p.v + b * p.sv.b + hk * p.sv.h;
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
            auto load = [&](const T* base, int d, int D, int64_t sd) {   // (what lies beyond Dk is cleared below, what lies beyond Dv not stored)
                if constexpr (WHOLE) return *(const V*)(base + (d < D ? d : 0));
                else return att_load<T>(base, d, D, sd, p.vec);
            };
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
            if (WHOLE && p.Dk < DP) {   // (an infinity among the keys must not meet the query's zeros)
#pragma unroll
                for (int u = 0; u < NS; u++)
#pragma unroll
                    for (int i = 0; i < NT; i++)
                        if (GN * i + h * N >= p.Dk) ka[u][i] = 0;
            }
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
    if (live) att_store<AttOps<A, DP>>(p, o, head, b, hk, row, split, h, m, l);   // (E = N there, too: the same elements in the same accumulators)
}

// Joins the shares of each row, first their weights across the lanes, then lanes along the width: a wavefront per row or, with many shares, the
// four of a workgroup, whose sums are added in order.  A launch and two dependent reads: 4.4 us for 256 rows of 32 shares (a wavefront each 5.5).
// One query of a long sequence needs many shares: 100 000 keys of 2 heads at width 64 take 37 us with 256 shares, 101 us with 64.
constexpr uint32_t kMaxShares = 256;
template <class A, bool WIDE>
__global__ __launch_bounds__(256) void attention_join_kernel(AttArgs<typename A::T> p) {
    using T = typename A::T;
    __shared__ T weights[4][kMaxShares];
    __shared__ T sums[4][128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t row = WIDE ? blockIdx.x : (size_t)blockIdx.x * 4 + wave;
    if (row >= (size_t)p.B * p.Hk * p.rows) return;   // (a whole workgroup or, with no barrier below, a wavefront)
    const uint32_t head = (uint32_t)(row / p.rows), r = (uint32_t)(row - (size_t)head * p.rows);
    const int b = head / p.Hk, hk = head - b * p.Hk;
    constexpr int K = kMaxShares / 64;
    T pm[K], pl[K], m = -(T)__builtin_inf(), l = 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const uint32_t s = k * 64 + lane;
        pm[k] = s < p.splits ? p.part_m[row * p.splits + s] : -(T)__builtin_inf();
        pl[k] = s < p.splits ? p.part_l[row * p.splits + s] : T(0);
    }
#pragma unroll
    for (int k = 0; k < K; k++) m = pm[k] > m ? pm[k] : m;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T y = __shfl_xor(m, d);
        m = y > m ? y : m;
    }
    const T mu = m == -(T)__builtin_inf() ? T(0) : m;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const T w = A::exp_(pm[k] - mu);              // (0 beyond the last share)
        weights[wave][k * 64 + lane] = w;
        l += w * pl[k];
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
    wave_lds_fence();                                 // (a wavefront uses its own weights only)
    const T f = l == T(0) ? T(0) : T(1) / l;
    T* orow = p.o + att_row(p, p.so, b, hk, r);
    const T* part = p.part_o + row * p.splits * p.Dv;
    for (int d = lane; d < p.Dv; d += 64) {
        T o = 0;
#pragma unroll 8
        for (uint32_t s = WIDE ? wave : 0; s < p.splits; s += WIDE ? 4 : 1) o += weights[wave][s] * part[(size_t)s * p.Dv + d];
        if (WIDE) sums[wave][d] = o;
        else orow[d * p.so.d] = o * f;
    }
    if (WIDE) {
        __syncthreads();
        for (int d = threadIdx.x; d < p.Dv; d += 256) orow[d * p.so.d] = (((sums[0][d] + sums[1][d]) + sums[2][d]) + sums[3][d]) * f;
    }
    if (p.lse_out && lane == 0 && (!WIDE || wave == 0)) p.lse_out[att_row(p, p.slse, b, hk, r)] = att_lse_of<A>(m, l);
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------------
// delta[row] = sum_d d_out out, 16 lanes a row, summed in 64 bits and rounded once.  Bound by its bytes: 32 768 rows of 128 (34 MB) in 7 us.
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

// dS scales with what is upstream and may lie far below the numbers it is made of.  Cut in three parts it therefore carries a factor 2^64 until dq
// and dk are stored: without it a part falls under bf16's least denormal, 2^-133, from dS = 2^-110 down.  Where that factor overflows, the
// sums are not finite.
template <class Ops> constexpr typename Ops::T kAttUp = std::is_empty<typename Ops::Watch>::value ? 1 : 18446744073709551616.0;
template <class Ops> __device__ __forceinline__ typename Ops::T att_ds(typename Ops::T prob, typename Ops::T dp_delta, typename Ops::T scale_up) {
    return kAttUp<Ops> == 1 ? prob * dp_delta * scale_up : prob * scale_up * dp_delta;
}
constexpr int kGradWaves = 4;
template <class Ops> struct GradLds {
    typename Ops::Tile a[2], b[2];
    typename Ops::T lse[2][kAttTile], delta[2][kAttTile];
    uint32_t words[kAttWords];
};

// dq: a wavefront owns M rows and walks the keys, as the forward pass does.
template <class Ops>
__device__ __forceinline__ bool att_dq(const AttArgs<typename Ops::T>& p, GradLds<Ops>& lds, uint32_t at) {
    using A = typename Ops::Mma;
    using T = typename A::T;
    using Acc = typename A::Acc;
    constexpr int M = A::M, NS = kAttTile / M, ND = Ops::ND, WAVES = kGradWaves;
    uint32_t head, inner;
    att_place(at, p.blocks * p.splits, p.B * p.Hk, &head, &inner);
    const uint32_t block = inner / p.splits, split = inner - block * p.splits;
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (M - 1), h = lane / M;
    const uint32_t row = (block * WAVES + wave) * M + c;
    const bool live = row < p.rows;
    typename Ops::Watch watch;
    typename Ops::Operand q, g;
    Ops::load(q, p.q + att_row(p, p.sq, b, hk, live ? row : 0), p.Dk, p.sq.d, p.vec, h, watch);
    Ops::load(g, p.d_out + att_row(p, p.sdo, b, hk, live ? row : 0), p.Dv, p.sdo.d, p.vec, h, watch);
    const T lse = live ? att_lse<A>(p.lse[att_row(p, p.slse, b, hk, row)]) : (T)__builtin_inf();
    const T delta = live ? p.delta[(size_t)head * p.rows + row] : T(0);
    const T scale_up = p.scale * kAttUp<Ops>;
    Acc dq[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) dq[i] = 0;
    const int tiles = (p.Lk + kAttTile - 1) / kAttTile;
    const int t0 = split * p.split_tiles, t1 = tiles < (int)(t0 + p.split_tiles) ? tiles : (int)(t0 + p.split_tiles);
    const T* kb = p.k + b * p.sk.b + hk * p.sk.h;
    const T* vb = p.v + b * p.sv.b + hk * p.sv.h;
    typename Ops::Stage st;
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
            }, p.Dk, p.Dv, p.sk.d, p.sv.d, p.vec);
        };
        int i = next(0), buf = 0;
        if (i < wn) fetch(i);
        while (i < wn) {
            const uint32_t word = __builtin_amdgcn_readfirstlane(lds.words[i]);
            Ops::store(st, lds.a[buf], lds.b[buf], p.Dk, p.Dv, word, watch);
            __syncthreads();
            i = next(i + 1);
            if (i < wn) fetch(i);
#pragma unroll
            for (int u = 0; u < NS; u++) {
                Acc s, dp;
                Ops::scores(s, lds.a[buf], q, dp, lds.b[buf], g, u, c, h);
#pragma unroll
                for (int r = 0; r < A::R; r++) s[r] = att_ds<Ops>(A::exp_(s[r] * p.scale_base - lse), dp[r] - delta, scale_up);
                if (word != ~0u) {
#pragma unroll
                    for (int r = 0; r < A::R; r++)
                        if (!((word >> (u * M + A::acc_row(r, h))) & 1u)) s[r] = 0;
                }
                Ops::outer(dq, lds.a[buf], s, u, c, h);
            }
            buf ^= 1;
        }
    }
    if (!std::is_empty<typename Ops::Watch>::value && __syncthreads_or((int)(Ops::failed(watch) || (live && !att_finite<Ops>(dq))))) return false;
    if (!live) return true;
    T* o;
    int64_t sd;
    if (p.splits == 1) {
        o = p.dq + att_row(p, p.sdq, b, hk, row);
        sd = p.sdq.d;
    } else {
        o = p.part_dq + (((size_t)split * p.B * p.Hk + head) * p.rows + row) * p.Dk;
        sd = 1;
    }
    Ops::put(o, sd, p.Dk, dq, T(1) / kAttUp<Ops>, h);
    return true;
}

// dk and dv: a wavefront owns M keys and walks the rows of the group's query heads.
template <class Ops>
__device__ __forceinline__ bool att_dkv(const AttArgs<typename Ops::T>& p, GradLds<Ops>& lds, uint32_t at) {
    using A = typename Ops::Mma;
    using T = typename A::T;
    using Acc = typename A::Acc;
    constexpr int M = A::M, NS = kAttTile / M, ND = Ops::ND, WAVES = kGradWaves;
    uint32_t head, inner;
    att_place(at, p.kblocks * p.ksplits, p.B * p.Hk, &head, &inner);
    const uint32_t block = inner / p.ksplits, split = inner - block * p.ksplits;
    const int b = head / p.Hk, hk = head - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (M - 1), h = lane / M;
    const int key = (block * WAVES + wave) * M + c;
    const bool in = key < p.Lk, on = att_key_on(p, b, key);
    typename Ops::Watch watch, of_mine;
    typename Ops::Operand k, v;
    Ops::load(k, p.k + b * p.sk.b + hk * p.sk.h + (in ? key : 0) * p.sk.l, p.Dk, p.sk.d, p.vec, h, of_mine);
    Ops::load(v, p.v + b * p.sv.b + hk * p.sv.h + (in ? key : 0) * p.sv.l, p.Dv, p.sv.d, p.vec, h, of_mine);
    if (on) {
        watch = of_mine;
    } else {
        Ops::clear(k);
        Ops::clear(v);
    }
    Acc dk[ND], dv[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) dk[i] = dv[i] = 0;
    const int tiles = ((int)p.rows + kAttTile - 1) / kAttTile;
    const int t0 = split * p.ksplit_tiles, t1 = tiles < (int)(t0 + p.ksplit_tiles) ? tiles : (int)(t0 + p.ksplit_tiles);
    const bool any = __syncthreads_or((int)on);   // a block whose keys are all masked has nothing to add up
    const T scale_up = p.scale * kAttUp<Ops>;
    typename Ops::Stage st;
    T lse = 0, delta = 0;                          // of row threadIdx.x of the tile in flight
    auto fetch = [&](int t) {
        const uint32_t r0 = (uint32_t)t * kAttTile;
        st.load([&](int r, int which) {
            const uint32_t at_row = r0 + r < p.rows ? r0 + r : p.rows - 1;
            return which ? p.d_out + att_row(p, p.sdo, b, hk, at_row) : p.q + att_row(p, p.sq, b, hk, at_row);
        }, p.Dk, p.Dv, p.sq.d, p.sdo.d, p.vec);
        if (threadIdx.x < kAttTile) {
            const uint32_t r = r0 + threadIdx.x;
            const uint32_t at_row = r < p.rows ? r : p.rows - 1;   // (rows beyond the last are zeros in the tile: what they get here adds nothing)
            lse = p.lse[att_row(p, p.slse, b, hk, at_row)];         // as loaded: computing with it here would wait for the whole tile
            delta = p.delta[(size_t)head * p.rows + at_row];
        }
    };
    int buf = 0;
    if (any && t0 < t1) fetch(t0);
    for (int t = t0; any && t < t1; t++) {
        const uint32_t left = p.rows - (uint32_t)t * kAttTile;
        Ops::store(st, lds.a[buf], lds.b[buf], p.Dk, p.Dv, left >= 32 ? ~0u : (1u << left) - 1u, watch);
        if (threadIdx.x < kAttTile) {
            lds.lse[buf][threadIdx.x] = t * kAttTile + threadIdx.x < p.rows ? att_lse<A>(lse) : (T)__builtin_inf();
            lds.delta[buf][threadIdx.x] = delta;
        }
        __syncthreads();
        if (t + 1 < t1) fetch(t + 1);
#pragma unroll
        for (int u = 0; u < NS; u++) {
            Acc s, dp;
            Ops::scores(s, lds.a[buf], k, dp, lds.b[buf], v, u, c, h);
#pragma unroll
            for (int r = 0; r < A::R; r++) {
                const int i = u * M + A::acc_row(r, h);
                const T pr = A::exp_(s[r] * p.scale_base - lds.lse[buf][i]);   // (a key that is off adds up something, too, which is dropped below)
                dp[r] = att_ds<Ops>(pr, dp[r] - lds.delta[buf][i], scale_up);
                s[r] = pr;
            }
            Ops::outer(dv, lds.b[buf], s, dk, lds.a[buf], dp, u, c, h);
        }
        buf ^= 1;
    }
    if (!std::is_empty<typename Ops::Watch>::value && __syncthreads_or((int)(Ops::failed(watch) || (on && !(att_finite<Ops>(dk) && att_finite<Ops>(dv)))))) return false;
    if (!in) return true;
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
    if (!on) {
#pragma unroll
        for (int i = 0; i < ND; i++) dk[i] = dv[i] = 0;
    }
    Ops::put(ok, sk, p.Dk, dk, T(1) / kAttUp<Ops>, h);
    Ops::put(ov, sv, p.Dv, dv, T(1), h);
    return true;
}

// Both halves of the backward pass in one launch, so that neither leaves compute units idle while the other runs out: `first` workgroups of
// dq (dq_first) or of dk and dv, then those of the other.  The half with the longer walks goes first: what is left for the end is short.
// Bound as the forward pass, with seven products of a tile instead of two (S and dP are computed in both halves: dS kept by
// one for the other would be memory of rows x keys): 4 x 16 heads, 512 queries, 1024 keys at width 128 in 323 us with the launch for delta (float instructions: 493 us), 16 x 16 heads
// at width 64 in 550 to 580 us (910 to 930 us).  At width 96 and 128 one wavefront a SIMD has no other to hide its vector instructions behind.
template <class A, int DP, bool WHOLE>
__global__ __launch_bounds__(64 * kGradWaves, DP <= 64 ? 2 : 1) void attention_grad_kernel(AttArgs<typename A::T> p, uint32_t first, bool dq_first) {
    using First = typename AttFirst<A, DP, kGradWaves, WHOLE>::Ops;
    using Exact = AttOps<A, DP, kGradWaves, WHOLE>;
    __shared__ union {
        GradLds<First> first;
        GradLds<Exact> exact;
    } lds;
    const bool front = blockIdx.x < first;
    const uint32_t at = front ? blockIdx.x : blockIdx.x - first;
    if (front == dq_first) {
        if constexpr (!std::is_same<First, Exact>::value)
            if (!p.exact && att_dq(p, lds.first, at)) return;
        att_dq(p, lds.exact, at);
    } else {
        if constexpr (!std::is_same<First, Exact>::value)
            if (!p.exact && att_dkv(p, lds.first, at)) return;
        att_dkv(p, lds.exact, at);
    }
}

// Adds up the shares in their order: workgroups [0, kv) take rows of dk and dv, the others rows of dq; a thread per element.  4 us where shares
// are few rows' (2 x 2 heads, 231 rows, 333 keys of 40 doubles).
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
// Up to here the kernel without LDS (two blocks of 16 rows read the keys twice, the second time from the L2).  It against the tiles, in us: 2000 keys of
// 64 heads at width 64, 16 rows 20 and 34, 32 rows 25 and 34, 33 rows 35 and 34, 64 rows 36 and 36, 96 rows 57 and 35; 1500 keys of 256 heads 32 rows 50
// and 73, 64 rows 112 and 78; 200 keys of 128 heads 32 rows 15 and 17, 64 rows 20 and 20; at width 128 (2000 keys of 64 heads) 32 rows 47 and 83, 64
// rows 73 and 85.  Double precision, 16 rows 34 and 45, 32 rows 47 and 47, 33 rows 58 and 56 (64 heads).
constexpr int64_t kFewRows = 32;

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

// Estimates in microseconds that choose the numbers of shares, fitted to 512 queries and 1024 keys at widths 32 to 128: a 32-row tile costs a
// wavefront 0.0105 us a product and column in single precision and 0.0145 in double precision (matrix instructions, and what cutting, staging and
// softmax leave uncovered), and 0.3 or 1 us besides; starting and ending a workgroup 4 us.  Up to padded width 64 two workgroups of
// four wavefronts fit a compute unit (they share the pipes), above one.  With shares chosen so, with as many as make 256 workgroups, and with none, in us: 300
// queries over 3000 keys of 4 heads at width 128 35, 35 and 290, their gradient 81, 111 and 322; 40 queries over 60 000 keys of 2 heads 35, 48 and 3827;
// 33 over 2000 of 64 heads 34, 48 and 150; 513 over 2000 of 16 heads 46, 54 and 110; 1000 x 1000 of 8 heads 31, 31 and 58, their gradient 64, 62 and 128.
inline int att_resident(int64_t width) { return width <= 64 ? 2 : 1; }
template <class T> double att_walk_us(int64_t width, int products, int64_t tiles) {
    const double padded = (double)((width + 31) / 32 * 32), column = sizeof(T) == 4 ? 0.0105 : 0.0145, tile = sizeof(T) == 4 ? 0.3 : 1.0;
    return 4.0 + tiles * (products * padded * column * att_resident(width) + tile);
}
// `n` workgroups of `each` us on `slots` places: what a place has to do on average, and half a walk for the uneven end
inline double att_span_us(double n, double each, double slots) { return n <= slots ? each : n * each / slots + 0.5 * each; }
inline double att_join_us(double bytes) { return bytes > 0 ? 5.0 + 2 * bytes / 4.0e6 : 0.0; }
// Most memory for the parts of a walk that is shared: 256 MB, which the Infinity Cache holds between the two launches.  A walk that would
// need more has workgroups enough to fill the chip many times over, and its uneven end costs it little.
constexpr double kAttPartBytes = 256.0 * 1024 * 1024;

struct AttPlan {
    int waves;   // 0: the kernel for few rows
    uint32_t blocks, splits, split_tiles;
    size_t o_bytes, m_bytes, total;
};
// The shares depend on the larger width alone, so that the memory they need for Dk = Dv = width is enough for every smaller one.
template <class T> AttPlan att_plan(int64_t heads, int64_t rows, int64_t Lk, int64_t Dk, int64_t Dv) {
    constexpr int M = MmaOf<T>::Tile::M;
    AttPlan p;
    const int64_t width = Dk > Dv ? Dk : Dv;
    const int64_t tiles = (Lk + kAttTile - 1) / kAttTile;
    if (rows <= kFewRows) {
        p.waves = 0;
        p.blocks = cdiv(rows, 16);
        att_shares(heads * p.blocks, tiles, 8 * kAttCUs, kMaxShares, &p.splits, &p.split_tiles);    // two wavefronts per SIMD
    } else {
        p.waves = rows <= 2 * M ? 2 : 4;
        p.blocks = cdiv(rows, (int64_t)p.waves * M);
        const double slots = (double)kAttCUs * att_resident(width) * 4 / p.waves;
        double best = 0;
        for (int64_t n = 1; n <= kMaxShares && (n == 1 || 2 * n <= tiles + 1); n += n < 16 ? 1 : n / 8) {
            const int64_t each = (tiles + n - 1) / n;
            const double bytes = n > 1 ? (double)heads * rows * n * width * sizeof(T) : 0.0;
            const double us = att_span_us((double)heads * p.blocks * n, att_walk_us<T>(width, 2, each), slots) + att_join_us(bytes);
            if (n > 1 && (us >= best || bytes > kAttPartBytes)) continue;
            best = us;
            p.split_tiles = (uint32_t)(each < 1 ? 1 : each);
            p.splits = cdiv(tiles, p.split_tiles);
            if (p.splits < 1) p.splits = 1;
        }
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
    // both numbers of shares at once: the halves run side by side (more than 64 gave nothing: 57 us, 60 us with up to 256, for 30 000 keys)
    const int64_t width = Dk > Dv ? Dk : Dv, tk = (Lk + kAttTile - 1) / kAttTile, tr = (rows + kAttTile - 1) / kAttTile;
    const double slots = (double)kAttCUs * att_resident(width), qn = (double)heads * p.blocks, kn = (double)heads * p.kblocks;
    double best = 0;
    for (int64_t n = 1; n <= 64 && (n == 1 || 2 * n <= tk + 1); n = n < 8 ? n + 1 : n + n / 4)
        for (int64_t k = 1; k <= 64 && (k == 1 || 2 * k <= tr + 1); k = k < 8 ? k + 1 : k + k / 4) {
            const int64_t eq = (tk + n - 1) / n, ek = (tr + k - 1) / k;
            const double uq = att_walk_us<T>(width, 3, eq), uk = att_walk_us<T>(width, 4, ek), longest = uq > uk ? uq : uk;
            const double even = (qn * n * uq + kn * k * uk) / slots + 0.5 * (uq < uk ? uq : uk);
            const double bytes = ((n > 1 ? (double)heads * rows * n : 0.0) + (k > 1 ? (double)heads * Lk * 2 * k : 0.0)) * width * sizeof(T);
            const double us = (qn * n + kn * k <= slots || even < longest ? longest : even) + att_join_us(bytes);
            if ((n > 1 || k > 1) && (us >= best || bytes > kAttPartBytes)) continue;
            best = us;
            p.split_tiles = (uint32_t)(eq < 1 ? 1 : eq);
            p.splits = cdiv(tk, p.split_tiles);
            if (p.splits < 1) p.splits = 1;
            p.ksplit_tiles = (uint32_t)(ek < 1 ? 1 : ek);
            p.ksplits = cdiv(tr, p.ksplit_tiles);
            if (p.ksplits < 1) p.ksplits = 1;
        }
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
    const AttPlan pl = att_plan<T>(heads, p.rows, p.Lk, p.Dk, p.Dv);
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
        if (width <= 64 && p.whole) hipLaunchKernelGGL((attention_few_kernel<Few, 64, true>), grid, dim3(64), 0, s, p);
        else if (width <= 64) hipLaunchKernelGGL((attention_few_kernel<Few, 64, false>), grid, dim3(64), 0, s, p);
        else if (p.whole) hipLaunchKernelGGL((attention_few_kernel<Few, 128, true>), grid, dim3(64), 0, s, p);
        else hipLaunchKernelGGL((attention_few_kernel<Few, 128, false>), grid, dim3(64), 0, s, p);
    } else {
        att_widths<T>(width, [&](auto dp) {
            if constexpr (2 * Tile::M > kFewRows) {   // (else two wavefronts have no more rows than the kernel for few takes)
                if (pl.waves == 2) {
                    if (p.whole) hipLaunchKernelGGL((attention_kernel<Tile, dp.value, 2, true>), grid, dim3(128), 0, s, p);
                    else hipLaunchKernelGGL((attention_kernel<Tile, dp.value, 2, false>), grid, dim3(128), 0, s, p);
                    return;
                }
            }
            if (p.whole) hipLaunchKernelGGL((attention_kernel<Tile, dp.value, 4, true>), grid, dim3(256), 0, s, p);
            else hipLaunchKernelGGL((attention_kernel<Tile, dp.value, 4, false>), grid, dim3(256), 0, s, p);
        });
    }
    DNH_LAUNCH_CHECK();
    if (p.splits > 1) {
        if (p.splits > 16) hipLaunchKernelGGL((attention_join_kernel<Tile, true>), dim3(heads * p.rows), dim3(256), 0, s, p);
        else hipLaunchKernelGGL((attention_join_kernel<Tile, false>), dim3(cdiv((int64_t)heads * p.rows, 4)), dim3(256), 0, s, p);
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
    // a tile costs three products in dq, four in dk and dv
    const bool dq_first = 3 * (int64_t)p.split_tiles >= 4 * (int64_t)p.ksplit_tiles;
    const uint32_t first = dq_first ? dq : kv;
    att_widths<T>(p.Dk > p.Dv ? p.Dk : p.Dv, [&](auto dp) {
        if (p.whole) hipLaunchKernelGGL((attention_grad_kernel<Tile, dp.value, true>), dim3(kv + dq), dim3(64 * kGradWaves), 0, s, p, first, dq_first);
        else hipLaunchKernelGGL((attention_grad_kernel<Tile, dp.value, false>), dim3(kv + dq), dim3(64 * kGradWaves), 0, s, p, first, dq_first);
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
