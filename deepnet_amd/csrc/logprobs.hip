// dnh_token_log_probs, dnh_token_log_probs_grad: from a model's logits, per row of length V,
//
//   lse      = log sum_j e^{x_j}                 log_prob = x_token - lse
//   entropy  = lse - sum_j p_j x_j               p_j      = e^{x_j - lse}
//   top      = the K largest logits as log probabilities with their indices, ties to the lower index
//
// and for upstream gradients g of log_prob and h of entropy
//
//   d_j = g (1[j = token] - p_j) - h p_j (log p_j + entropy)
//
// All of it in one pass over the logits: with m the maximum so far, s = sum e^{x - m} and a = sum e^{x - m} (x - m) are rescaled when
// m grows, lse = m + log s and entropy = log s - a / s.  Bound by HBM: the forward pass reads R x V, the gradient reads and writes it.
#include "model_ops.h"

using namespace dnh;

namespace {

constexpr int kBlock = 256, kWaves = kBlock / 64;
constexpr int kMaxTop = 64;                     // one alternative per lane of a wavefront
constexpr uint32_t kNoIndex = 0xFFFFFFFFu;
constexpr int kSlice = 4096;                    // a row is shared among no more workgroups than have this many elements, but for the last one's rest

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896340736f); }
__device__ __forceinline__ double exp_of(double d) { return exp(d); }
template <class T> __device__ __forceinline__ T neg_inf() { return -(T)__builtin_inf(); }
// e^d d vanishes with e^d, also for an element that cannot be chosen (d = -inf) or lies so far down that s d would overflow: the factor
// is held at a value where e^d has vanished
__device__ __forceinline__ float entropy_factor(float d) { return fmaxf(d, -1.0e4f); }
__device__ __forceinline__ double entropy_factor(double d) { return fmax(d, -1.0e6); }

// Running statistics of part of a row.  The sums are kept in 64 bits: with one dominant logit s = 1 + (the rest), and the entropy is
// made of the rest.
struct Stats {
    double m, s, a;
};
__device__ __forceinline__ Stats no_stats() { return Stats{-__builtin_inf(), 0.0, 0.0}; }
__device__ __forceinline__ Stats merge(const Stats& x, const Stats& y) {
    if (x.m == -__builtin_inf() && x.s == 0.0) return y;
    if (y.m == -__builtin_inf() && y.s == 0.0) return x;
    const Stats &hi = x.m >= y.m ? x : y, &lo = x.m >= y.m ? y : x;
    const double d = entropy_factor(lo.m - hi.m), e = exp(d);
    return Stats{hi.m, hi.s + lo.s * e, hi.a + e * (lo.a + lo.s * d)};
}
__device__ __forceinline__ Stats wave_merge(Stats x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        Stats y{__shfl_xor(x.m, d), __shfl_xor(x.s, d), __shfl_xor(x.a, d)};
        x = merge(x, y);
    }
    return x;
}

// ---- the best K of a stream, one per lane in descending order ---------------------------------------------------------------------
template <class T> __device__ __forceinline__ bool better(T v, uint32_t i, T w, uint32_t j) { return v > w || (v == w && i < j); }

// Lane moves on 32-bit words, element-wise for wider types: no LDS round trip, which a cross-lane shuffle would take.
template <class X> __device__ __forceinline__ X read_lane(X x, int lane) {   // lane: the same for the whole wavefront
    int w[sizeof(X) / 4];
    __builtin_memcpy(w, &x, sizeof(X));
#pragma unroll
    for (int k = 0; k < (int)(sizeof(X) / 4); k++) w[k] = __builtin_amdgcn_readlane(w[k], lane);
    __builtin_memcpy(&x, w, sizeof(X));
    return x;
}
template <class X> __device__ __forceinline__ X from_lane_below(X x) {       // lane l gets lane l - 1's, lane 0 keeps its own
    int w[sizeof(X) / 4];
    __builtin_memcpy(w, &x, sizeof(X));
#pragma unroll
    for (int k = 0; k < (int)(sizeof(X) / 4); k++) w[k] = __builtin_amdgcn_update_dpp(w[k], w[k], 0x138, 0xf, 0xf, false);   // wave_shr:1
    __builtin_memcpy(&x, w, sizeof(X));
    return x;
}

// Where a wavefront spreads some lanes' elements over all lanes.
template <class T> struct Spread {
    T x[64];
    uint32_t first[64], taken[64];
};

template <class T> struct TopList {
    T v;             // the lane-th best so far
    uint32_t i;      // kNoIndex: none yet
    T floor_v;       // the K-th best
    uint32_t floor_i;
    __device__ __forceinline__ void clear() {
        v = neg_inf<T>();
        i = kNoIndex;
        // The floor lives in scalar registers, and a double there must not be a constant the compiler knows: it then writes -inf with one
        // 64-bit scalar move, whose literal has only 32 bits (ROCm 7.2: the register pair gets 0.0).
        int w[sizeof(T) / 4];
        __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
        for (int k = 0; k < (int)(sizeof(T) / 4); k++) asm volatile("" : "+s"(w[k]));
        __builtin_memcpy(&floor_v, w, sizeof(T));
        floor_i = kNoIndex;
    }
    // every lane offers one element (`in`: it has one); NaN is never better than anything
    __device__ __forceinline__ void offer(T x, uint32_t j, bool in, int K) {
        unsigned long long m = __ballot(in && better(x, j, floor_v, floor_i));
        const int lane = threadIdx.x & 63;
        while (m) {
            const int src = __builtin_ctzll(m);
            const T cv = read_lane(x, src);
            const uint32_t ci = read_lane(j, src);
            const int at = __popcll(__ballot(better(v, i, cv, ci)));
            const T pv = from_lane_below(v);
            const uint32_t pi = from_lane_below(i);
            v = lane > at ? pv : lane == at ? cv : v;
            i = lane > at ? pi : lane == at ? ci : i;
            floor_v = read_lane(v, K - 1);
            floor_i = read_lane(i, K - 1);
            // the floor has risen: those still waiting have to pass it anew
            m &= m - 1;
            m &= __ballot(better(x, j, floor_v, floor_i));
        }
    }
    // joins another list of the same order.  Position by position the better one of this list and the other one reversed are the best
    // 64 of both, descending and then ascending or the other way round; six exchanges sort them.
    __device__ __forceinline__ void join(T ov, uint32_t oi, int K) {
        const int lane = threadIdx.x & 63;
        const T rv = __shfl(ov, 63 - lane);
        const uint32_t ri = __shfl(oi, 63 - lane);
        if (better(rv, ri, v, i)) {
            v = rv;
            i = ri;
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) exchange(v, i, d, (lane & d) == 0);
        floor_v = read_lane(v, K - 1);
        floor_i = read_lane(i, K - 1);
    }
    // one step of a sorting network: of lanes that differ in bit d, those with `keep` keep the better element
    static __device__ __forceinline__ void exchange(T& v, uint32_t& i, int d, bool keep) {
        const T pv = __shfl_xor(v, d);
        const uint32_t pi = __shfl_xor(i, d);
        if (better(pv, pi, v, i) == keep) {
            v = pv;
            i = pi;
        }
    }
    // C elements of every lane, element c with index first + step(c) (ascending), those from index `end` on missing; big: the largest of them.
    // When many lanes hold something for the list, as at the start of a row, the lanes' largest elements are sorted and joined at once; the
    // K-th of them is then a floor that few others pass.  Then, 64 / C at a time, the lanes whose largest element reaches the floor spread
    // their elements over the wavefront, and those above the floor are inserted one by one.
    template <int C, class Step>
    __device__ __forceinline__ void offer_all(const T (&x)[C], T big, uint32_t first, Step step, uint32_t end, int K, Spread<T>& sp) {
        unsigned long long m = __ballot(big >= floor_v);
        if (m == 0) return;
        const int lane = threadIdx.x & 63;
        uint32_t taken = kNoIndex;
        if (__popcll(m) > 8) {
            T bv = x[0];
            uint32_t bi = first + step(0);
#pragma unroll
            for (int c = 1; c < C; c++)
                if (x[c] > bv || bv != bv) {
                    bv = x[c];
                    bi = first + step(c);
                }
            if (bv != bv || bi >= end) {                 // a lane of NaNs, or of missing elements (-inf), has nothing to offer
                bv = neg_inf<T>();
                bi = kNoIndex;
            }
            taken = bi;
#pragma unroll
            for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
                for (int d = k >> 1; d; d >>= 1) exchange(bv, bi, d, ((lane & d) == 0) == ((lane & k) == 0));
            join(bv, bi, K);
            m = __ballot(big >= floor_v);
        }
        constexpr int L = 64 / C;                        // lanes that spread at a time
        while (m) {
            const int rank = __popcll(m & ((1ull << lane) - 1ull));
            if (((m >> lane) & 1ull) && rank < L) {
#pragma unroll
                for (int c = 0; c < C; c++) sp.x[rank * C + c] = x[c];
                sp.first[rank] = first;
                sp.taken[rank] = taken;
            }
            wave_lds_fence();
            const uint32_t j = sp.first[lane / C] + step(lane % C);
            const T v_lane = sp.x[lane];
            const uint32_t taken_lane = sp.taken[lane / C];
            wave_lds_fence();                            // (the next lanes' elements go to the same places)
            offer(v_lane, j, lane / C < __popcll(m) && j < end && j != taken_lane, K);
#pragma unroll
            for (int k = 0; k < L; k++) m &= m - 1;      // (0 stays 0)
            m &= __ballot(big >= floor_v);
        }
    }
};

// ---- forward --------------------------------------------------------------------------------------------------------------------------
template <class T> struct LogProbArgs {
    const T* x;                  // logits
    int64_t xd;                  // their stride along the vocabulary
    int64_t vocab;
    RowPlan<7> rp;               // rows of: logits, tokens, log_probs, lse, entropy, top values, top tokens
    const int64_t* tokens;       // any of these may be missing
    T *log_probs, *lse, *entropy, *top_v;
    int64_t* top_i;
    int64_t top_vd, top_id;
    int K;
    int32_t* err;
};

// Writes a row's results; every lane of one wavefront calls it, lane i holding the i-th alternative.
template <class T>
__device__ __forceinline__ void finish_row(const LogProbArgs<T>& p, uint32_t row, const Stats& st, T top_v, uint32_t top_i) {
    const int lane = threadIdx.x & 63;
    int64_t off[7];
    row_offsets(p.rp, row, off);
    const bool empty = st.m == -__builtin_inf() && st.s == 0.0;   // every logit is -inf: nothing can be chosen
    const double log_s = empty ? 0.0 : log(st.s);
    if (lane == 0) {
        if (p.lse) p.lse[off[3]] = (T)(empty ? -__builtin_inf() : st.m + log_s);
        if (p.entropy) p.entropy[off[4]] = (T)(empty ? 0.0 : log_s - st.a / st.s);
        if (p.tokens) {
            const int64_t tok = p.tokens[off[1]];
            if (tok >= 0 && tok < p.vocab) p.log_probs[off[2]] = empty ? neg_inf<T>() : (T)(((double)p.x[off[0] + tok * p.xd] - st.m) - log_s);
            else *p.err = 1;
        }
    }
    if (lane < p.K) {
        p.top_v[off[5] + lane * p.top_vd] = top_i == kNoIndex ? (T)__builtin_nan("") : empty ? neg_inf<T>() : (T)(((double)top_v - st.m) - log_s);
        p.top_i[off[6] + lane * p.top_id] = top_i == kNoIndex ? DNH_NOT_FOUND : (int64_t)top_i;
    }
}

// One element into a thread's running statistics, m already at least its value.
template <class T> __device__ __forceinline__ void take(T x, T m, double& s, double& a) {
    const T d = x - m, e = exp_of(d);
    s += (double)e;
    a += (double)(e * entropy_factor(d));
}
// the larger one; of a number and a quiet NaN the number (the instruction makes a NaN of a number and a signaling one)
__device__ __forceinline__ float larger(float x, float y) {
    float r;
    // (fmaxf first quiets both operands: three instructions.  The operands must not come straight from a transcendental instruction, whose
    // result the compiler separates from its user by a wait state only where it knows the user.)
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(x), "v"(y));
    return r;
}
__device__ __forceinline__ double larger(double x, double y) { return y > x || x != x ? y : x; }

// U x N elements at once.  Single precision is bound by instructions if every term goes to double precision by itself (28 cycles of 4 per
// element, 155 us for 4096 rows of 50 048 without alternatives, against 127 us as it is), so groups of U x N are added up in 32 bits first, five roundings
// deep.  That would lose the rest beside a dominant logit, whose term is exactly 1: the ones are kept out of the sum (v_fract_f32 turns 1
// into 0 and leaves what is below 1) and counted by the difference of the sums with and without them, which is a whole number
// up to a rounding.
template <int U, int N> __device__ __forceinline__ void take_all(const float (&x)[U][N], float m, double& s, double& a) {
    float below[N], all[N], ed[N];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float d = x[u][e] - m, t = exp_of(d), f = larger(d, -1.0e4f);   // (as entropy_factor)
            below[e] = u ? below[e] + __builtin_amdgcn_fractf(t) : __builtin_amdgcn_fractf(t);
            all[e] = u ? all[e] + t : t;
            ed[e] = u ? __builtin_fmaf(t, f, ed[e]) : t * f;
        }
#pragma unroll
    for (int w = 1; w < N; w <<= 1)
#pragma unroll
        for (int e = 0; e + w < N; e += 2 * w) {
            below[e] += below[e + w];
            all[e] += all[e + w];
            ed[e] += ed[e + w];
        }
    s += (double)below[0] + (double)__builtin_rintf(all[0] - below[0]);
    a += (double)ed[0];
}
template <int U, int N> __device__ __forceinline__ void take_all(const double (&x)[U][N], double m, double& s, double& a) {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < N; e++) take(x[u][e], m, s, a);
}
// e^d for the sums' rescaling.  Single precision: the fraction of the exponent on the fast instruction (2 u), the whole part exactly; the
// library's double-precision exponential would keep 20 registers of constants alive through the loop.
__device__ __forceinline__ double shrink(double d, float) {
    const double t = d * 1.44269504088896340736, n = __builtin_rint(t);
    return ldexp((double)__builtin_amdgcn_exp2f((float)(t - n)), (int)n);
}
__device__ __forceinline__ double shrink(double d, double) { return exp(d); }

// A workgroup takes elements [j0, j1) of a row.  With one workgroup per row it writes the results, else its statistics and list.
// Without alternatives it runs at the memory's rate: 4096 rows of 50 048 floats (820 MB) in 127 us, 6.5 TB/s.  With 5 alternatives 149 to 152 us: sorting
// the start of a row and inserting what passes the floor later take turns with the loads of the same wavefront.  One row of 128 000 with 20
// alternatives is a chain of latencies: 32 slices in 11 us, joined in 9 us.
template <class T, bool VEC, bool TOP>
__global__ __launch_bounds__(kBlock, TOP ? 5 : 1) void log_probs_kernel(LogProbArgs<T> p, uint32_t splits, uint32_t slice, Stats* __restrict__ part_st, T* __restrict__ part_v,
                                                           uint32_t* __restrict__ part_i) {
    constexpr int N = VEC ? kVecN<T> : 1, U = 4;
    using V = typename Vec16<T>::type;
    const uint32_t row = blockIdx.x / splits, split = blockIdx.x - row * splits;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t off[7];
    row_offsets(p.rp, row, off);
    const T* x = p.x + off[0];
    const int64_t j0 = (int64_t)split * slice, j1 = p.vocab - j0 < slice ? p.vocab : j0 + slice;
    // the wavefront's maximum, and each lane's sums relative to it: with one maximum for all lanes, sums are rescaled (a double-precision
    // exponential) about three times a row instead of in nearly every step, and lanes are joined by additions
    T m = neg_inf<T>();
    double s = 0, a = 0;
    __shared__ Spread<T> spread[TOP ? kWaves : 1];
    TopList<T> top;
    top.clear();
    for (int64_t j = j0; j < j1; j += U * kBlock * N) {
        T v[U][N];
        const T* xs = x + j * p.xd;                                                 // the same for the whole workgroup
        const int mine = (int)threadIdx.x * N, left = j1 - j < U * kBlock * N ? (int)(j1 - j) : U * kBlock * N;
        if (left == U * kBlock * N) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                if constexpr (VEC) {
                    const V w = __builtin_nontemporal_load((const V*)(xs + (mine + u * kBlock * N)));
#pragma unroll
                    for (int e = 0; e < N; e++) v[u][e] = w[e];
                } else {
                    v[u][0] = xs[(mine + u * kBlock) * p.xd];
                }
            }
        } else {
            // (a missing element has probability 0)
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int at = mine + u * kBlock * N;
                if (VEC && at + N <= left) {
                    const V w = *(const V*)(xs + at);
#pragma unroll
                    for (int e = 0; e < N; e++) v[u][e] = w[e % kVecN<T>];
                } else {
#pragma unroll
                    for (int e = 0; e < N; e++) v[u][e] = at + e < left ? xs[VEC ? (int64_t)(at + e) : (at + e) * p.xd] : neg_inf<T>();
                }
            }
        }
        T big = neg_inf<T>();                                                       // of the numbers; NaN of either kind is passed over
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < N; e++) big = v[u][e] > big ? v[u][e] : big;
        if (__ballot(big > m)) {
            T to = big > m ? big : m;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) to = larger(to, __shfl_xor(to, d));
            const double d = entropy_factor((double)m - (double)to), e = shrink(d, T());   // (m = -inf: the sums are still zero)
            a = e * (a + s * d);
            s *= e;
            m = to;
        }
        take_all(v, m == neg_inf<T>() ? T(0) : m, s, a);
        if constexpr (TOP) {
            T flat[U * N];
#pragma unroll
            for (int k = 0; k < U * N; k++) flat[k] = v[k / N][k % N];
            top.offer_all(flat, big, (uint32_t)j + (uint32_t)mine, [](int k) { return (uint32_t)(k / N * kBlock * N + k % N); }, (uint32_t)j1, p.K, spread[wave]);
        }
    }
    // the wavefronts' parts meet in LDS; the first wavefront joins them
    __shared__ Stats wst[kWaves];
    __shared__ T wv[kWaves][kMaxTop];
    __shared__ uint32_t wi[kWaves][kMaxTop];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        s += __shfl_xor(s, d);
        a += __shfl_xor(a, d);
    }
    const Stats mine{(double)m, s, a};
    if (lane == 0) wst[wave] = mine;
    if constexpr (TOP) {
        wv[wave][lane] = top.v;
        wi[wave][lane] = top.i;
    }
    __syncthreads();
    if (wave != 0) return;
    Stats all = mine;
    for (int w = 1; w < kWaves; w++) {
        all = merge(all, wst[w]);
        if constexpr (TOP) top.join(wv[w][lane], wi[w][lane], p.K);
    }
    if (splits == 1) {
        finish_row(p, row, all, top.v, top.i);
        return;
    }
    if (lane == 0) part_st[blockIdx.x] = all;
    if (TOP && lane < p.K) {
        part_v[(size_t)blockIdx.x * p.K + lane] = top.v;
        part_i[(size_t)blockIdx.x * p.K + lane] = top.i;
    }
}

// Joins the parts of a shared row: the wavefronts of a workgroup take parts in turn, then each other's lists two by two.
constexpr int kJoinWaves = 16;
template <class T>
__global__ __launch_bounds__(64 * kJoinWaves) void log_probs_join_kernel(LogProbArgs<T> p, uint32_t splits, const Stats* __restrict__ part_st,
                                                                         const T* __restrict__ part_v, const uint32_t* __restrict__ part_i) {
    __shared__ T wv[kJoinWaves][kMaxTop];
    __shared__ uint32_t wi[kJoinWaves][kMaxTop];
    const uint32_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool mine = lane < p.K;
    TopList<T> top;
    top.clear();
    if (p.K > 0) {
        for (uint32_t k = wave; k < splits; k += kJoinWaves) {
            const size_t at = ((size_t)row * splits + k) * p.K + lane;
            top.join(mine ? part_v[at] : neg_inf<T>(), mine ? part_i[at] : kNoIndex, p.K);
        }
        for (int half = kJoinWaves / 2; half; half >>= 1) {
            if (wave >= half && wave < 2 * half) {
                wv[wave][lane] = top.v;
                wi[wave][lane] = top.i;
            }
            __syncthreads();
            if (wave < half) top.join(wv[wave + half][lane], wi[wave + half][lane], p.K);
        }
    }
    if (wave != 0) return;
    Stats st = no_stats();
    for (uint32_t k = lane; k < splits; k += 64) st = merge(st, part_st[(size_t)row * splits + k]);
    st = wave_merge(st);
    finish_row(p, row, st, top.v, top.i);
}

// Workgroups that share a row.  A workgroup per row fills the chip from about two rows per compute unit on; below that the rows are cut
// into slices, one for each kSlice elements at most and all of about one length, until there are about four workgroups per compute unit.
constexpr uint32_t kCUs = 256;   // MI355X; a constant, so that the size of the scratch memory can be asked for without a device
uint32_t split_count(uint32_t rows, int64_t vocab) {
    const int64_t want = (4 * kCUs + rows - 1) / rows, most = (vocab + kSlice - 1) / kSlice;
    if (rows >= 2 * kCUs || most <= 1) return 1;
    return (uint32_t)(want < most ? want : most);
}

struct PartPlan {
    uint32_t splits, slice;
    size_t st_bytes, v_bytes, i_bytes, total;
};
PartPlan part_plan(uint32_t rows, int64_t vocab, int K, int esize) {
    PartPlan p;
    p.splits = split_count(rows, vocab);
    const int64_t per = (vocab + p.splits - 1) / p.splits;
    p.slice = (uint32_t)((per + 255) / 256 * 256);   // (a multiple of 256 elements: slices of an aligned row start aligned)
    p.splits = (uint32_t)((vocab + p.slice - 1) / p.slice);
    if (p.splits < 1) p.splits = 1;
    const size_t parts = (size_t)rows * p.splits;
    p.st_bytes = up256(parts * sizeof(Stats));
    p.v_bytes = up256(parts * K * esize);
    p.i_bytes = up256(parts * K * 4);
    p.total = p.splits == 1 ? 0 : p.st_bytes + p.v_bytes + p.i_bytes;
    return p;
}

template <class T>
int32_t log_probs(const DnhTensor* log_probs, const DnhTensor* lse, const DnhTensor* entropy, const DnhTensor* top_v, const DnhTensor* top_i,
                  const DnhTensor* logits, const DnhTensor* tokens, uint32_t rows, int K, void* scratch, size_t scratch_bytes, hipStream_t s) {
    const int nd = logits->ndims - 1;
    LogProbArgs<T> p;
    p.x = (const T*)elem_ptr(logits);
    p.xd = logits->stride[nd];
    p.vocab = logits->shape[nd];
    auto or_logits = [&](const DnhTensor* t) { return t ? t : logits; };
    p.rp = make_row_plan<7>(nd, {logits, or_logits(tokens), or_logits(log_probs), or_logits(lse), or_logits(entropy), or_logits(top_v), or_logits(top_i)});
    p.tokens = tokens ? (const int64_t*)elem_ptr(tokens) : nullptr;
    p.log_probs = log_probs ? (T*)elem_ptr(log_probs) : nullptr;
    p.lse = lse ? (T*)elem_ptr(lse) : nullptr;
    p.entropy = entropy ? (T*)elem_ptr(entropy) : nullptr;
    p.top_v = top_v ? (T*)elem_ptr(top_v) : nullptr;
    p.top_i = top_i ? (int64_t*)elem_ptr(top_i) : nullptr;
    p.top_vd = top_v ? top_v->stride[nd] : 0;
    p.top_id = top_i ? top_i->stride[nd] : 0;
    p.K = K;
    p.err = nullptr;
    if (tokens) DNH_TRY(error_flag_ptr(s, &p.err));
    const PartPlan pp = part_plan(rows, p.vocab, K, (int)sizeof(T));
    char* ws = nullptr;
    WorkspaceLease lease;
    DNH_TRY(get_scratch(s, pp.total, scratch, scratch_bytes, (void**)&ws, lease, "dnh_token_log_probs"));
    Stats* st = (Stats*)ws;
    T* pv = (T*)(ws + pp.st_bytes);
    uint32_t* pi = (uint32_t*)(ws + pp.st_bytes + pp.v_bytes);
    const bool vec = p.xd == 1;
    const dim3 grid(rows * pp.splits), block(kBlock);
    if (vec && K) hipLaunchKernelGGL((log_probs_kernel<T, true, true>), grid, block, 0, s, p, pp.splits, pp.slice, st, pv, pi);
    else if (vec) hipLaunchKernelGGL((log_probs_kernel<T, true, false>), grid, block, 0, s, p, pp.splits, pp.slice, st, pv, pi);
    else if (K) hipLaunchKernelGGL((log_probs_kernel<T, false, true>), grid, block, 0, s, p, pp.splits, pp.slice, st, pv, pi);
    else hipLaunchKernelGGL((log_probs_kernel<T, false, false>), grid, block, 0, s, p, pp.splits, pp.slice, st, pv, pi);
    DNH_LAUNCH_CHECK();
    if (pp.splits > 1) {
        hipLaunchKernelGGL((log_probs_join_kernel<T>), dim3(rows), dim3(K ? 64 * kJoinWaves : 64), 0, s, p, pp.splits, (const Stats*)st, (const T*)pv, (const uint32_t*)pi);
        DNH_LAUNCH_CHECK();
    }
    return DNH_OK;
}

// ---- gradient ---------------------------------------------------------------------------------------------------------------------------
template <class T> struct GradArgs {
    T* d;
    const T* x;
    int64_t dd, xd, vocab;
    RowPlan<7> rp;    // rows of: d_logits, logits, tokens, lse, entropy, d_log_probs, d_entropy
    const int64_t* tokens;
    const T *lse, *entropy, *g, *h;   // entropy and h may be missing together
    uint32_t slices;
    int32_t* err;
};

template <class T, bool ENT>
__device__ __forceinline__ T grad_of(T x, T lse, T H, T g, T h) {
    const T lp = x - lse, p = exp_of(lp);
    if constexpr (ENT) return -(p * (g + h * (entropy_factor(lp) + H)));
    else return -(g * p);
}

// A workgroup takes U x 16 bytes per thread of a row, straight through: 4096 rows of 50 048 floats are read and written (1.64 GB) in 265 us,
// 6.2 TB/s, what a copy reaches.  Double precision is bound by its exponential: 333 rows of 32 003 in 31 us, 5.6 TB/s of 171 MB from the cache.
template <class T, bool VEC, bool ENT>
__global__ __launch_bounds__(kBlock) void log_probs_grad_kernel(GradArgs<T> p) {
    constexpr int N = VEC ? kVecN<T> : 1, U = 4;
    using V = typename Vec16<T>::type;
    const uint32_t row = blockIdx.x / p.slices, slice = blockIdx.x - row * p.slices;
    int64_t off[7];
    row_offsets(p.rp, row, off);
    const int64_t tok = p.tokens[off[2]];
    if (!(tok >= 0 && tok < p.vocab)) {
        if (slice == 0 && threadIdx.x == 0) *p.err = 1;
        return;
    }
    const T lse = p.lse[off[3]], g = p.g[off[5]];
    T H = 0, h = 0;
    if constexpr (ENT) {
        H = p.entropy[off[4]];
        h = p.h[off[6]];
    }
    const bool empty = lse == neg_inf<T>();   // nothing can be chosen in this row: its gradient is zero
    const T* x = p.x + off[1];
    T* d = p.d + off[0];
    const int64_t j0 = (int64_t)slice * (U * kBlock * N) + threadIdx.x * N;
    auto one = [&](T v, int64_t j) {
        if (empty) return T(0);
        const T r = grad_of<T, ENT>(v, lse, H, g, h);
        return j == tok ? r + g : r;
    };
    if (VEC && (int64_t)(slice + 1) * (U * kBlock * N) <= p.vocab) {
        V v[U];
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = __builtin_nontemporal_load((const V*)(x + j0 + u * kBlock * N));
#pragma unroll
        for (int u = 0; u < U; u++) {
            V r;
#pragma unroll
            for (int e = 0; e < N; e++) r[e] = one(v[u][e], j0 + u * kBlock * N + e);
            __builtin_nontemporal_store(r, (V*)(d + j0 + u * kBlock * N));
        }
        return;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
        for (int e = 0; e < N; e++) {
            const int64_t j = j0 + u * kBlock * N + e;
            if (j < p.vocab) d[j * p.dd] = one(x[j * p.xd], j);
        }
}

template <class T>
int32_t log_probs_grad(const DnhTensor* d, const DnhTensor* x, const DnhTensor* tokens, const DnhTensor* lse, const DnhTensor* entropy, const DnhTensor* g,
                       const DnhTensor* h, uint32_t rows, hipStream_t s) {
    const int nd = x->ndims - 1;
    GradArgs<T> p;
    p.d = (T*)elem_ptr(d);
    p.x = (const T*)elem_ptr(x);
    p.dd = d->stride[nd];
    p.xd = x->stride[nd];
    p.vocab = x->shape[nd];
    p.rp = make_row_plan<7>(nd, {d, x, tokens, lse, entropy ? entropy : lse, g, h ? h : g});
    p.tokens = (const int64_t*)elem_ptr(tokens);
    p.lse = (const T*)elem_ptr(lse);
    p.entropy = entropy ? (const T*)elem_ptr(entropy) : nullptr;
    p.g = (const T*)elem_ptr(g);
    p.h = h ? (const T*)elem_ptr(h) : nullptr;
    DNH_TRY(error_flag_ptr(s, &p.err));
    const bool vec = p.dd == 1 && p.xd == 1;
    p.slices = cdiv(p.vocab, (int64_t)4 * kBlock * (vec ? kVecN<T> : 1));
    if ((int64_t)rows * p.slices > (1 << 24) - 1) return fail(DNH_ERR_NOT_SUPPORTED, "dnh_token_log_probs_grad: more than 2^24 workgroups of work");
    const dim3 grid(rows * p.slices), block(kBlock);
    if (vec && h) hipLaunchKernelGGL((log_probs_grad_kernel<T, true, true>), grid, block, 0, s, p);
    else if (vec) hipLaunchKernelGGL((log_probs_grad_kernel<T, true, false>), grid, block, 0, s, p);
    else if (h) hipLaunchKernelGGL((log_probs_grad_kernel<T, false, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((log_probs_grad_kernel<T, false, false>), grid, block, 0, s, p);
    DNH_LAUNCH_CHECK();
    return DNH_OK;
}

// logits [i_1 .. i_n; V]
int32_t check_logits(const DnhTensor* x, const char* what, uint32_t* rows) {
    DNH_TRY(check_tensor(x, what));
    DNH_TRY(check_float(x, x->dtype, what, "logits"));
    if (x->ndims < 1) return fail(DNH_ERR_INVALID_ARG, "%s: logits need a last axis of alternatives", what);
    if (x->shape[x->ndims - 1] > 0x7FFFFFFF) return fail(DNH_ERR_NOT_SUPPORTED, "%s: rows of more than 2^31 - 1 logits", what);
    return count_rows(x, x->ndims - 1, what, rows);
}
// one value per row
int32_t check_per_row(const DnhTensor* t, const DnhTensor* x, int32_t dtype, const char* what, const char* name) {
    DNH_TRY(check_tensor(t, what));
    if (t->dtype != dtype) return fail(DNH_ERR_INVALID_ARG, "%s: %s is %s, not %s", what, name, dtype_name(t->dtype), dtype_name(dtype));
    if (t->ndims != x->ndims - 1 || !same_leading(t, x, x->ndims - 1))
        return fail(DNH_ERR_INVALID_ARG, "%s: %s must have the logits' shape without its last axis", what, name);
    return DNH_OK;
}
int32_t check_row_target(const DnhTensor* t, const DnhTensor* x, const char* what, const char* name) {
    DNH_TRY(check_target(t, what, name));
    return check_per_row(t, x, x->dtype, what, name);
}

}  // namespace

extern "C" int32_t dnh_token_log_probs_scratch_bytes(int32_t dtype, int64_t rows, int64_t vocab, int64_t top, size_t* bytes) {
    if (!bytes || !dtype_is_fp(dtype) || rows < 0 || rows > 0x7FFFFFFF || vocab < 0 || vocab > 0x7FFFFFFF || top < 0 || top > kMaxTop)
        return fail(DNH_ERR_INVALID_ARG, "dnh_token_log_probs_scratch_bytes: bad argument");
    *bytes = rows && vocab ? part_plan((uint32_t)rows, vocab, (int)top, dtype_size(dtype)).total : 0;
    return DNH_OK;
}

extern "C" int32_t dnh_token_log_probs(const DnhTensor* log_probs_t, const DnhTensor* lse, const DnhTensor* entropy, const DnhTensor* top_log_probs,
                                       const DnhTensor* top_tokens, const DnhTensor* logits, const DnhTensor* tokens, void* scratch, size_t scratch_bytes,
                                       void* stream) {
    const char* what = "dnh_token_log_probs";
    uint32_t rows;
    DNH_TRY(check_logits(logits, what, &rows));
    const int nd = logits->ndims - 1;
    if (!tokens != !log_probs_t) return fail(DNH_ERR_INVALID_ARG, "%s: tokens and log_probs are given together or not at all", what);
    if (!top_log_probs != !top_tokens) return fail(DNH_ERR_INVALID_ARG, "%s: top_log_probs and top_tokens are given together or not at all", what);
    if (!log_probs_t && !lse && !entropy && !top_tokens) return fail(DNH_ERR_INVALID_ARG, "%s: nothing to compute", what);
    if (tokens) {
        DNH_TRY(check_per_row(tokens, logits, DNH_I64, what, "tokens"));
        DNH_TRY(check_row_target(log_probs_t, logits, what, "log_probs"));
    }
    if (lse) DNH_TRY(check_row_target(lse, logits, what, "lse"));
    if (entropy) DNH_TRY(check_row_target(entropy, logits, what, "entropy"));
    int K = 0;
    if (top_tokens) {
        DNH_TRY(check_target(top_log_probs, what, "top_log_probs"));
        DNH_TRY(check_target(top_tokens, what, "top_tokens"));
        if (top_log_probs->dtype != logits->dtype || top_tokens->dtype != DNH_I64)
            return fail(DNH_ERR_INVALID_ARG, "%s: top_log_probs must be %s and top_tokens int64", what, dtype_name(logits->dtype));
        if (top_tokens->ndims != nd + 1 || !same_leading(top_tokens, logits, nd) || !same_shape(top_log_probs, top_tokens))
            return fail(DNH_ERR_INVALID_ARG, "%s: top_log_probs and top_tokens must have the logits' shape with the last axis cut to the number of alternatives", what);
        const int64_t k = top_tokens->shape[nd];
        if (k > logits->shape[nd]) return fail(DNH_ERR_INVALID_ARG, "%s: %lld alternatives of %lld logits", what, (long long)k, (long long)logits->shape[nd]);
        if (k > kMaxTop) return fail(DNH_ERR_NOT_SUPPORTED, "%s: more than %d alternatives", what, kMaxTop);
        K = (int)k;
    }
    if (rows == 0) return DNH_OK;
    if (logits->shape[nd] == 0) return fail(DNH_ERR_INVALID_ARG, "%s: rows without logits", what);
    if (rows > (1u << 24) - 1) return fail(DNH_ERR_NOT_SUPPORTED, "%s: more than 2^24 - 1 rows", what);
    DNH_TRY(check_apart<7>({log_probs_t, lse, entropy, top_log_probs, top_tokens, logits, tokens},
                           {"log_probs", "lse", "entropy", "top_log_probs", "top_tokens", "logits", "tokens"}, 5, what));
    DNH_TRY(ensure_init());
    return logits->dtype == DNH_F32 ? log_probs<float>(log_probs_t, lse, entropy, top_log_probs, top_tokens, logits, tokens, rows, K, scratch, scratch_bytes, (hipStream_t)stream)
                                    : log_probs<double>(log_probs_t, lse, entropy, top_log_probs, top_tokens, logits, tokens, rows, K, scratch, scratch_bytes, (hipStream_t)stream);
}

extern "C" int32_t dnh_token_log_probs_grad(const DnhTensor* d_logits, const DnhTensor* logits, const DnhTensor* tokens, const DnhTensor* lse,
                                            const DnhTensor* entropy, const DnhTensor* d_log_probs, const DnhTensor* d_entropy, void* stream) {
    const char* what = "dnh_token_log_probs_grad";
    uint32_t rows;
    DNH_TRY(check_logits(logits, what, &rows));
    DNH_TRY(check_target(d_logits, what, "d_logits"));
    if (d_logits->dtype != logits->dtype || !same_shape(d_logits, logits)) return fail(DNH_ERR_INVALID_ARG, "%s: d_logits must have the logits' type and shape", what);
    if (!entropy != !d_entropy) return fail(DNH_ERR_INVALID_ARG, "%s: entropy and d_entropy are given together or not at all", what);
    DNH_TRY(check_per_row(tokens, logits, DNH_I64, what, "tokens"));
    DNH_TRY(check_per_row(lse, logits, logits->dtype, what, "lse"));
    DNH_TRY(check_per_row(d_log_probs, logits, logits->dtype, what, "d_log_probs"));
    if (entropy) {
        DNH_TRY(check_per_row(entropy, logits, logits->dtype, what, "entropy"));
        DNH_TRY(check_per_row(d_entropy, logits, logits->dtype, what, "d_entropy"));
    }
    if (rows == 0 || logits->shape[logits->ndims - 1] == 0) return DNH_OK;
    DNH_TRY(check_apart<7>({d_logits, same_view(d_logits, logits) ? nullptr : logits, tokens, lse, entropy, d_log_probs, d_entropy},
                           {"d_logits", "logits", "tokens", "lse", "entropy", "d_log_probs", "d_entropy"}, 1, what));
    DNH_TRY(ensure_init());
    return logits->dtype == DNH_F32 ? log_probs_grad<float>(d_logits, logits, tokens, lse, entropy, d_log_probs, d_entropy, rows, (hipStream_t)stream)
                                    : log_probs_grad<double>(d_logits, logits, tokens, lse, entropy, d_log_probs, d_entropy, rows, (hipStream_t)stream);
}
