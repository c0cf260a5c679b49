// dnh_embedding, dnh_embedding_grad: rows of a table by token number, scaled, and the gradient of the table.
//
//   t[i, :]       = scale * table[tokens[i], :]
//   d_table[v, :] = scale * sum over { i : tokens[i] = v } of d_out[i, :]      (the sum in 64 bits, in an order that depends on the tokens alone; one rounding)
//
// Both are bound by HBM: the lookup reads every row it names and writes N x D, the gradient reads N x D and writes V x D.
// The gradient needs no atomics: the N token numbers are sorted (stable, with their positions) and each run of equal tokens is added up
// by one thread per column vector, so the result has the same bits on every run; few tokens are compared with each other instead.
#include "model_ops.h"

using namespace dnh;

namespace {

constexpr int kBlock = 256;

// ---- lookup ---------------------------------------------------------------------------------------------------------------------
// 2^txl threads share a row (16 bytes each), U rows per thread in flight.  Bound by HBM: 65 536 rows of 1024 floats from a table of 50 000 are
// read (rows named twice come from the caches) and written in 59 us, 268 MB of stores alone at 4.6 TB/s; 16 rows take 2.8 us, one
// memory round trip for the token and one for its row.
template <class T, bool VEC, int U>
__global__ __launch_bounds__(kBlock) void embedding_kernel(T* __restrict__ t, const T* __restrict__ table, const int64_t* __restrict__ tokens,
                                                           RowPlan<2> rp, uint32_t n, int64_t td, int64_t tab_row, int64_t tab_d, int64_t vocab,
                                                           int64_t width, T scale, int txl, int32_t* err) {
    constexpr int N = VEC ? kVecN<T> : 1;
    using V = typename Vec16<T>::type;
    const int sub = threadIdx.x >> txl, lane = threadIdx.x & ((1 << txl) - 1), per = kBlock >> txl;
    const int64_t c = ((int64_t)blockIdx.y << txl | lane) * N;
    if (c >= width) return;
    int64_t toff[U], tok[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t i = (blockIdx.x * U + u) * per + sub;
        ok[u] = i < n;
        int64_t off[2] = {0, 0};
        if (ok[u]) row_offsets(rp, i, off);
        toff[u] = off[0];
        tok[u] = ok[u] ? tokens[off[1]] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
        if (ok[u] && !(tok[u] >= 0 && tok[u] < vocab)) {
            *err = 1;
            ok[u] = false;
        }
    if (VEC && c + N <= width) {
        V v[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (ok[u]) v[u] = *(const V*)(table + tok[u] * tab_row + c);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (ok[u]) __builtin_nontemporal_store(v[u] * scale, (V*)(t + toff[u] + c));
    } else {
        for (int64_t e = c; e < c + N && e < width; e++)
#pragma unroll
            for (int u = 0; u < U; u++)
                if (ok[u]) t[toff[u] + e * td] = table[tok[u] * tab_row + e * tab_d] * scale;
    }
}

template <class T, bool VEC>
int32_t launch_embedding(const DnhTensor* t, const DnhTensor* table, const DnhTensor* tokens, uint32_t n, T scale, hipStream_t s, int32_t* err) {
    const int nd = tokens->ndims;
    const int64_t width = table->shape[1];
    const RowPlan<2> rp = make_row_plan<2>(nd, {t, tokens});
    const int64_t items = VEC ? (width + kVecN<T> - 1) / kVecN<T> : width;
    const int txl = lanes_log2(items), per = kBlock >> txl;
    const unsigned gy = cdiv(items, (int64_t)1 << txl);
    // four rows per thread once the rows alone fill the chip; one where that would leave compute units idle
    const bool deep = (int64_t)cdiv(n, per * 4) * gy >= 2 * device_cus();
    const dim3 grid(cdiv(n, per * (deep ? 4 : 1)), gy);
    if (grid.x >= 1u << 24) return fail(DNH_ERR_NOT_SUPPORTED, "dnh_embedding: %u rows of %lld elements are more than one call can address", n, (long long)width);
#define ARGS (T*)elem_ptr(t), (const T*)elem_ptr(table), (const int64_t*)elem_ptr(tokens), rp, n, t->stride[nd], table->stride[0], table->stride[1], \
             table->shape[0], width, scale, txl, err
    if (deep) hipLaunchKernelGGL((embedding_kernel<T, VEC, 4>), grid, dim3(kBlock), 0, s, ARGS);
    else hipLaunchKernelGGL((embedding_kernel<T, VEC, 1>), grid, dim3(kBlock), 0, s, ARGS);
#undef ARGS
    DNH_LAUNCH_CHECK();
    return DNH_OK;
}

// ---- sorting the tokens ------------------------------------------------------------------------------------------------------------
// Stable least-significant-digit radix sort of (token, position).  A token outside the table gets the key `vocab` and ends up behind
// all others, where nothing reads it.  Ranks come from ballots: lanes of a wavefront that share a digit find each other with one ballot
// per digit bit; each wavefront counts its own digits in LDS while it walks its part of the tile in order.  Bound by latency (barriers and
// dependent LDS accesses), not by bytes: 4095 tokens of 14 bits take one launch of 13 us, 32 768 of 16 bits two pairs of 6 + 13 us, in which
// the target is cleared besides (205 MB).  Up to 8192 tokens one workgroup is faster than a pair of launches for each digit.
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kMinDigitBits = 6, kMaxDigitBits = 9, kMaxDigits = 1 << kMaxDigitBits;
constexpr uint32_t kSmallSort = 8192;    // tokens that one workgroup sorts in LDS, in one launch
constexpr uint32_t kSortTile = 1024;     // tokens of a workgroup's step in the passes through memory: one a thread, as its stores scatter over
                                         // as many cache lines and a compute unit serves one line a cycle (4096: 15 us a pass instead of 9)
constexpr int64_t kMaxGradTokens = (int64_t)1 << 27;   // keeps every grid of the gradient below 2^32 threads
constexpr uint32_t kMaxChunks = 128;     // workgroups of such a pass: every one of them adds up the counts of all

struct TokenSource {
    const int64_t* tokens;
    RowPlan<1> rp;
    uint32_t n, vocab;
    int32_t* err;
};
__device__ __forceinline__ uint32_t token_key(const TokenSource& s, uint32_t i) {
    int64_t off[1];
    row_offsets(s.rp, i, off);
    const int64_t tok = s.tokens[off[0]];
    if (tok >= 0 && tok < (int64_t)s.vocab) return (uint32_t)tok;
    *s.err = 1;
    return s.vocab;
}

// Counters of (digit, wavefront), a digit's 16 side by side in 17 words: lanes of a wavefront with different digits meet different banks.
constexpr int kCounters = kMaxDigits * (kSortWaves + 1);
__device__ __forceinline__ int counter(uint32_t digit, int wave) { return (int)digit * (kSortWaves + 1) + wave; }

// Rank of each of the thread's E keys (key e of lane l of wave w stands at w * 64 E + 64 e + l) among the wavefront's keys of the same
// digit; the wavefront's counts per digit are left in cnt.
template <int E>
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[E], const bool (&live)[E], int bits, uint32_t* cnt, uint32_t (&rank)[E]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int e = 0; e < E; e++) {
        unsigned long long peers = __ballot(live[e]);
        for (int b = 0; b < bits; b++) {
            const bool set = (digit[e] >> b) & 1u;
            const unsigned long long with = __ballot(set);
            peers &= set ? with : ~with;
        }
        const uint32_t before = (uint32_t)__popcll(peers & ((1ull << lane) - 1ull));
        // LDS accesses of one wavefront are served in order: every lane reads the count, then the first of each group raises it
        const int at = counter(digit[e], wave);
        const uint32_t old = live[e] ? __hip_atomic_load(&cnt[at], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) : 0u;
        rank[e] = old + before;
        if (live[e] && before == 0) __hip_atomic_store(&cnt[at], old + (uint32_t)__popcll(peers), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
}

// Exclusive scan of one value per thread; every thread of the workgroup calls it.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* wave_sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    if (lane == 63) wave_sum[wave] = x;
    __syncthreads();
    uint32_t base = lane < wave ? wave_sum[lane] : 0u;   // (16 wavefronts: the sums before this one lie in its first lanes)
#pragma unroll
    for (int d = 1; d < kSortWaves; d <<= 1) base += __shfl_xor(base, d);
    base = __shfl(base, 0);
    __syncthreads();
    return base + x - v;
}

// Turns the counters into where each (digit, wavefront) starts in the sorted tile: an exclusive scan in that order, digits / 64 counters
// (all of one digit) a thread.  Every thread of the workgroup calls it, with the counters complete; it ends with a barrier.
__device__ __forceinline__ void scan_counters(uint32_t* cnt, int bits, uint32_t* wave_sum) {
    const int per = (1 << bits) / 64;
    const int at = counter(threadIdx.x * per / kSortWaves, threadIdx.x * per % kSortWaves);
    uint32_t sum = 0;
    for (int k = 0; k < per; k++) sum += cnt[at + k];
    uint32_t run = block_scan(sum, wave_sum);
    for (int k = 0; k < per; k++) {
        const uint32_t c = cnt[at + k];
        cnt[at + k] = run;
        run += c;
    }
    __syncthreads();
}

// Fills rows [row0, row1) of a target with zeros; workgroup `wg` of `wgs`.
template <class T> struct ZeroRows {
    T* t;
    int64_t row_stride, d_stride, width, row0, row1;
};
template <class T>
__device__ __forceinline__ void zero_rows(const ZeroRows<T>& z, uint32_t wg, uint32_t wgs, int threads) {
    using V = typename Vec16<T>::type;
    constexpr int N = kVecN<T>;
    const V zero = 0;
    if (z.row_stride == z.width && z.d_stride == 1) {   // one contiguous run
        const int64_t n = (z.row1 - z.row0) * z.width, nv = n / N;
        T* p = z.t + z.row0 * z.width;
        for (int64_t i = (int64_t)wg * threads + threadIdx.x; i < nv; i += (int64_t)wgs * threads) __builtin_nontemporal_store(zero, (V*)(p + i * N));
        if (wg == 0 && (int)threadIdx.x < n - nv * N) p[nv * N + threadIdx.x] = T(0);
        return;
    }
    for (int64_t r = z.row0 + wg; r < z.row1; r += wgs)
        for (int64_t c = threadIdx.x; c < z.width; c += threads) z.t[r * z.row_stride + c * z.d_stride] = T(0);
}

// Workgroup 0 sorts up to 1024 E tokens in LDS; the others clear the target meanwhile.
template <class T, int E>
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(TokenSource src, int npass, int bits, uint32_t* __restrict__ keys, uint32_t* __restrict__ pos,
                                                                  ZeroRows<T> z) {
    if (blockIdx.x > 0) {
        zero_rows(z, blockIdx.x - 1, gridDim.x - 1, kSortThreads);
        return;
    }
    __shared__ uint32_t lk[kSortThreads * E];
    __shared__ uint16_t lp[kSortThreads * E];
    __shared__ uint32_t cnt[kCounters];
    __shared__ uint32_t wave_sum[kSortWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t n = src.n, base = wave * 64 * E + lane;
    uint32_t k[E], p[E];
    bool live[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        p[e] = base + 64 * e;
        live[e] = p[e] < n;
        k[e] = live[e] ? token_key(src, p[e]) : 0;
    }
    const uint32_t digits = 1u << bits;
    for (int pass = 0; pass < npass; pass++) {
        const int sh = pass * bits;
        for (uint32_t d = threadIdx.x; d < digits * (kSortWaves + 1); d += kSortThreads) cnt[d] = 0;
        __syncthreads();
        uint32_t digit[E], rank[E];
#pragma unroll
        for (int e = 0; e < E; e++) digit[e] = (k[e] >> sh) & (digits - 1);
        wave_ranks<E>(digit, live, bits, cnt, rank);
        __syncthreads();
        scan_counters(cnt, bits, wave_sum);
        if (pass == npass - 1) {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (live[e]) {
                    const uint32_t to = cnt[counter(digit[e], wave)] + rank[e];
                    keys[to] = k[e];
                    pos[to] = p[e];
                }
            return;
        }
#pragma unroll
        for (int e = 0; e < E; e++)
            if (live[e]) {
                const uint32_t to = cnt[counter(digit[e], wave)] + rank[e];
                lk[to] = k[e];
                lp[to] = (uint16_t)p[e];
            }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; e++)
            if (live[e]) {
                k[e] = lk[base + 64 * e];
                p[e] = lp[base + 64 * e];
            }
    }
}

// One pass through memory, first half: how many tokens of each chunk have each digit -> counts[digit][chunk].
// keys == nullptr: the first pass, which reads the tokens themselves.
template <class T>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(TokenSource src, const uint32_t* __restrict__ keys, int shift, int bits, uint32_t chunk,
                                                                  uint32_t nchunks, uint32_t* __restrict__ counts, ZeroRows<T> z) {
    if (blockIdx.x >= nchunks) {
        zero_rows(z, blockIdx.x - nchunks, gridDim.x - nchunks, kSortThreads);
        return;
    }
    __shared__ uint32_t hist[kMaxDigits];
    const uint32_t digits = 1u << bits;
    if (threadIdx.x < digits) hist[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t i0 = blockIdx.x * chunk, i1 = src.n - i0 < chunk ? src.n : i0 + chunk;
    for (uint32_t i = i0 + threadIdx.x; i < i1; i += kSortThreads) {
        const uint32_t k = keys ? keys[i] : token_key(src, i);
        atomicAdd(&hist[(k >> shift) & (digits - 1)], 1u);
    }
    __syncthreads();
    if (threadIdx.x < digits) counts[(size_t)blockIdx.x * digits + threadIdx.x] = hist[threadIdx.x];
}

// Second half: every chunk's tokens go to their places.  A workgroup finds where its share of each digit starts by adding up the
// counts of all chunks itself (one launch fewer than a scan of its own).
template <class T>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(TokenSource src, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, int shift,
                                                                  int bits, uint32_t chunk, uint32_t nchunks, const uint32_t* __restrict__ counts,
                                                                  uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out, ZeroRows<T> z) {
    if (blockIdx.x >= nchunks) {
        zero_rows(z, blockIdx.x - nchunks, gridDim.x - nchunks, kSortThreads);
        return;
    }
    constexpr int E = kSortTile / kSortThreads;
    __shared__ uint32_t cnt[kCounters];
    __shared__ uint32_t start[kMaxDigits];   // where the chunk's next key of each digit goes
    __shared__ uint32_t wave_sum[kSortWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t digits = 1u << bits;
    const uint32_t i0 = blockIdx.x * chunk, i1 = src.n - i0 < chunk ? src.n : i0 + chunk;
    uint32_t k[E], p[E];
    auto load = [&](uint32_t t0) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const uint32_t i = t0 + wave * 64 * E + 64 * e + lane;
            k[e] = i >= i1 ? 0u : keys ? keys[i] : token_key(src, i);
            p[e] = i >= i1 ? 0u : keys ? pos[i] : i;
        }
    };
    load(i0);                                // in flight while the counts are added up
    uint32_t total = 0, before = 0;
    if (threadIdx.x < digits)
#pragma unroll 8
        for (uint32_t c = 0; c < nchunks; c++) {
            const uint32_t v = counts[(size_t)c * digits + threadIdx.x];
            before += c < blockIdx.x ? v : 0u;
            total += v;
        }
    const uint32_t first = block_scan(total, wave_sum);
    if (threadIdx.x < digits) start[threadIdx.x] = first + before;
    for (uint32_t t0 = i0; t0 < i1; t0 += kSortTile) {
        for (uint32_t d = threadIdx.x; d < digits * (kSortWaves + 1); d += kSortThreads) cnt[d] = 0;
        if (t0 != i0) load(t0);
        uint32_t digit[E], rank[E];
        bool live[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            live[e] = t0 + wave * 64 * E + 64 * e + lane < i1;
            digit[e] = (k[e] >> shift) & (digits - 1);
        }
        __syncthreads();
        wave_ranks<E>(digit, live, bits, cnt, rank);
        __syncthreads();
        scan_counters(cnt, bits, wave_sum);
#pragma unroll
        for (int e = 0; e < E; e++)
            if (live[e]) {
                const uint32_t to = start[digit[e]] + cnt[counter(digit[e], wave)] - cnt[counter(digit[e], 0)] + rank[e];
                keys_out[to] = k[e];
                pos_out[to] = p[e];
            }
        __syncthreads();
        // (the last wavefront's start of a digit, and what it has of it itself, are where the next tile goes on)
        if (t0 + kSortTile < i1 && threadIdx.x < digits)
            start[threadIdx.x] += (threadIdx.x + 1 < digits ? cnt[counter(threadIdx.x + 1, 0)] : kSortTile) - cnt[counter(threadIdx.x, 0)];
        __syncthreads();
    }
}

// ---- adding up the runs --------------------------------------------------------------------------------------------------------------
// The sorted list is cut into pieces of R entries; 2^txl threads take a piece, 16 bytes of the row each, and add in 64 bits.  A run
// inside the piece goes straight to its row of the target.  The part of a run that began in an earlier piece goes to the piece's first
// partial, the part of a run that goes on behind it to its second one; the second kernel adds those.  Bound by the reads of d_out, a row at
// a time in the tokens' order, eight in flight: 32 768 x 1024 floats (134 MB, part of it from the 256 MB cache) in 32 us.
template <class T> struct GradTarget {
    T* t;
    int64_t row_stride, d_stride, width;
    double scale;
    int accumulate;
};
template <class T>
__device__ __forceinline__ void put(const GradTarget<T>& g, uint32_t row, int64_t c, double v) {
    T* p = g.t + (int64_t)row * g.row_stride + c * g.d_stride;
    const double x = v * g.scale;
    *p = g.accumulate ? (T)((double)*p + x) : (T)x;
}

template <class T, bool VEC>
__global__ __launch_bounds__(kBlock) void embedding_sum_kernel(GradTarget<T> tg, const T* __restrict__ g, RowPlan<1> gp, int64_t gd, const uint32_t* __restrict__ keys,
                                                               const uint32_t* __restrict__ pos, uint32_t n, uint32_t vocab, int txl, uint32_t R, uint32_t pieces,
                                                               int64_t pitch, double* __restrict__ partial) {
    constexpr int N = VEC ? kVecN<T> : 1, U = 8;
    using V = typename Vec16<T>::type;
    const int sub = threadIdx.x >> txl, lane = threadIdx.x & ((1 << txl) - 1), per = kBlock >> txl;
    const uint32_t piece = blockIdx.x * per + sub;
    const int64_t c = ((int64_t)blockIdx.y << txl | lane) * N;
    if (piece >= pieces || c >= tg.width) return;
    const int live = (int)(tg.width - c < N ? tg.width - c : N);
    const uint32_t i0 = piece * R, i1 = n - i0 < R ? n : i0 + R;
    double acc[N];
#pragma unroll
    for (int e = 0; e < N; e++) acc[e] = 0;
    uint32_t cur = keys[i0];
    bool began_before = i0 > 0 && keys[i0 - 1] == cur;
    auto to_partial = [&](int which) {
        for (int e = 0; e < live; e++) partial[((size_t)piece * 2 + which) * pitch + c + e] = acc[e];
    };
    auto to_row = [&]() {
        if (cur == vocab) return;
        if (VEC && live == N && tg.d_stride == 1) {
            V* p = (V*)(tg.t + (int64_t)cur * tg.row_stride + c);
            V v = 0;
            if (tg.accumulate) v = *p;
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = (T)((double)v[e] + acc[e] * tg.scale);
            *p = v;
        } else {
            for (int e = 0; e < live; e++) put(tg, cur, c + e, acc[e]);
        }
    };
    for (uint32_t i = i0; i < i1; i += U) {
        uint32_t k[U];
        T x[U][N];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t j = i + u < i1 ? i + u : i1 - 1;
            k[u] = keys[j];
            int64_t off[1];
            row_offsets(gp, pos[j], off);
            const T* p = g + off[0];
            if (VEC && live == N) {
                const V v = *(const V*)(p + c);
#pragma unroll
                for (int e = 0; e < N; e++) x[u][e] = v[e];
            } else {
#pragma unroll
                for (int e = 0; e < N; e++) x[u][e] = e < live ? p[(c + e) * gd] : T(0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i + u >= i1) break;
            if (k[u] != cur) {
                if (began_before) to_partial(0);
                else to_row();
                began_before = false;
                cur = k[u];
#pragma unroll
                for (int e = 0; e < N; e++) acc[e] = 0;
            }
#pragma unroll
            for (int e = 0; e < N; e++) acc[e] += (double)x[u][e];
        }
    }
    if (began_before) to_partial(0);
    else if (i1 < n && keys[i1] == cur) to_partial(1);
    else to_row();
}

// Runs that cross pieces.  The workgroups of the piece in which such a run begins add its partials: 256 columns each, the pieces dealt
// to four wavefronts, whose sums are added in order.  The longest run decides: token frequencies of 1 / rank, 32 768 tokens, 10 us.
constexpr int kJoinThreads = 256, kJoinWaves = kJoinThreads / 64, kJoinCols = 256;
template <class T>
__global__ __launch_bounds__(kJoinThreads) void embedding_join_kernel(GradTarget<T> tg, const uint32_t* __restrict__ keys, uint32_t n, uint32_t vocab, uint32_t R,
                                                                      uint32_t pieces, int64_t pitch, const double* __restrict__ partial) {
    typedef double D2 __attribute__((ext_vector_type(2)));
    const uint32_t piece = blockIdx.x, i0 = piece * R, i1 = n - i0 < R ? n : i0 + R;
    if (i1 >= n) return;
    const uint32_t key = keys[i1 - 1], after = keys[i1], head = keys[i0], before = i0 > 0 ? keys[i0 - 1] : vocab;
    if (key == vocab || after != key) return;                                 // no run goes on behind this piece
    if (head == key && before == key) return;                                 // one does, but it began earlier
    __shared__ double sums[kJoinWaves][kJoinCols];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t more = 0;                                                        // pieces that continue the run
    for (;;) {
        const uint32_t q = piece + 1 + more + lane;
        const unsigned long long m = __ballot(q < pieces && keys[(size_t)q * R] == key);
        if (m != ~0ull) {
            more += (uint32_t)__builtin_ctzll(~m);
            break;
        }
        more += 64;
    }
    // a lane takes columns 2 l, 2 l + 1 and those 128 further on; the pitch is even, so a pair that begins in the row exists in the partials
    const int64_t c0 = (int64_t)blockIdx.y * kJoinCols + 2 * lane, c1 = c0 + kJoinCols / 2;
    const int64_t r0 = c0 < tg.width ? c0 : 0, r1 = c1 < tg.width ? c1 : 0;
    D2 a0 = 0, a1 = 0;
#pragma unroll 8
    for (uint32_t q = wave; q <= more; q += kJoinWaves) {
        const double* p = partial + ((size_t)(piece + q) * 2 + (q == 0 ? 1 : 0)) * pitch;
        a0 += *(const D2*)(p + r0);
        a1 += *(const D2*)(p + r1);
    }
    *(D2*)&sums[wave][2 * lane] = a0;
    *(D2*)&sums[wave][kJoinCols / 2 + 2 * lane] = a1;
    __syncthreads();
    const int64_t c = (int64_t)blockIdx.y * kJoinCols + threadIdx.x;
    if (c < tg.width) {
        double v = 0;
        for (int w = 0; w < kJoinWaves; w++) v += sums[w][threadIdx.x];
        put(tg, key, c, v);
    }
}

// ---- few tokens -----------------------------------------------------------------------------------------------------------------------
// Up to kFewTokens everything in one launch, without a sort: each workgroup reads all the tokens.  Those of leader i add up the rows of the
// tokens equal to the i-th unless one before it is equal, 16 bytes of the row per lane, equal tokens dealt to four wavefronts whose sums
// are added in order.  The others clear blocks of rows, leaving out those that a leader writes.  Bound by latency: the tokens, the rows, the sums.
// 512 tokens into 10 007 rows of 300 floats 8.4 us against 16.3 us sorted (513 tokens), 16 tokens 7.5 us; into 50 000 rows of 1024 (205 MB to
// clear) 45 us against 48.5; into 500 rows of 2000, where the sums are most of it, 12.4 us against 15.6 (in double precision 16.1 against 15.6).
constexpr uint32_t kFewTokens = 512;
constexpr int kFillRows = 2048;   // most rows of a block that is cleared at once
constexpr size_t kFewScratch = 256;   // what the query answers for them: none of it is used, but a call with less than the query says is refused
bool few_tokens(int64_t n, int64_t width) { return n <= kFewTokens && n * width <= (1 << 28); }   // (a grid of fewer than 2^32 threads for any width)
template <class T, bool VEC>
__global__ __launch_bounds__(kBlock) void embedding_grad_few_kernel(GradTarget<T> tg, TokenSource src, const T* __restrict__ g, RowPlan<1> gp, int64_t gd, uint32_t chunks,
                                                                    uint32_t block_rows, int txl) {
    constexpr int N = VEC ? kVecN<T> : 1, U = 8, COLS = 64 * N, WAVES = kBlock / 64, PER = kFewTokens / WAVES;
    using V = typename Vec16<T>::type;
    __shared__ uint32_t keys[kFewTokens];
    __shared__ uint32_t list[kFewTokens];
    __shared__ uint32_t counts[WAVES];
    __shared__ uint32_t marks[kFillRows / 32];
    __shared__ double sums[WAVES][COLS];
    const uint32_t n = src.n;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t i = threadIdx.x; i < kFewTokens; i += kBlock) keys[i] = i < n ? token_key(src, i) : src.vocab;
    __syncthreads();
    if (blockIdx.x >= n * chunks) {
        const uint32_t wg = blockIdx.x - n * chunks, wgs = gridDim.x - n * chunks;
        const int per = kBlock >> txl, sub = threadIdx.x >> txl, col = threadIdx.x & ((1 << txl) - 1);
        constexpr int NZ = kVecN<T>;
        for (uint64_t r0 = (uint64_t)wg * block_rows; r0 < src.vocab; r0 += (uint64_t)wgs * block_rows) {
            if (threadIdx.x < kFillRows / 32) marks[threadIdx.x] = 0;
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < n; i += kBlock)
                if (keys[i] >= r0 && keys[i] < r0 + block_rows && keys[i] != src.vocab) atomicOr(&marks[(keys[i] - (uint32_t)r0) >> 5], 1u << ((keys[i] - (uint32_t)r0) & 31));
            __syncthreads();
            for (uint32_t r = sub; r < block_rows && r0 + r < src.vocab; r += per) {
                if ((marks[r >> 5] >> (r & 31)) & 1u) continue;
                T* row = tg.t + (int64_t)(r0 + r) * tg.row_stride;
                for (int64_t c = (int64_t)col * NZ; c < tg.width; c += (int64_t)NZ << txl) {
                    if (tg.d_stride == 1 && c + NZ <= tg.width) {
                        __builtin_nontemporal_store(V(0), (V*)(row + c));
                    } else {
                        for (int64_t e = c; e < c + NZ && e < tg.width; e++) row[e * tg.d_stride] = T(0);
                    }
                }
            }
            __syncthreads();
        }
        return;
    }
    const uint32_t leader = blockIdx.x / chunks, key = keys[leader];
    // the list of equal tokens, in order: each wavefront finds those of its quarter
    uint32_t at[PER / 64], mine = 0;
    bool is[PER / 64], before = false;
#pragma unroll
    for (int e = 0; e < PER / 64; e++) {
        const uint32_t j = wave * PER + e * 64 + lane;
        is[e] = j < n && keys[j] == key;
        before |= is[e] && j < leader;
        const unsigned long long m = __ballot(is[e]);
        at[e] = mine + (uint32_t)__popcll(m & ((1ull << lane) - 1ull));
        mine += (uint32_t)__popcll(m);
    }
    if (lane == 0) counts[wave] = mine;
    if (__syncthreads_or((int)(before || key == src.vocab))) return;   // an equal token before it, or none of the table
    uint32_t first = 0, total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        if (w < wave) first += counts[w];
        total += counts[w];
    }
#pragma unroll
    for (int e = 0; e < PER / 64; e++)
        if (is[e]) list[first + at[e]] = wave * PER + e * 64 + lane;
    __syncthreads();
    const int64_t c = (int64_t)(blockIdx.x - leader * chunks) * COLS + lane * N;
    const int live = c >= tg.width ? 0 : (int)(tg.width - c < N ? tg.width - c : N);
    double acc[N];
#pragma unroll
    for (int e = 0; e < N; e++) acc[e] = 0;
    for (uint32_t k = wave; k < total; k += U * WAVES) {
        T x[U][N];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t q = k + u * WAVES;
            int64_t off[1];
            row_offsets(gp, list[q < total ? q : total - 1], off);
            const T* p = g + off[0];
            if (VEC && live == N) {
                const V v = *(const V*)(p + c);
#pragma unroll
                for (int e = 0; e < N; e++) x[u][e] = v[e];
            } else {
#pragma unroll
                for (int e = 0; e < N; e++) x[u][e] = e < live ? p[(c + e) * gd] : T(0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (k + u * WAVES < total) {
#pragma unroll
                for (int e = 0; e < N; e++) acc[e] += (double)x[u][e];
            }
    }
#pragma unroll
    for (int e = 0; e < N; e++) sums[wave][lane * N + e] = acc[e];
    __syncthreads();
    if (wave != 0 || live == 0) return;
    const int others = total < (uint32_t)WAVES ? (int)total : WAVES;
    for (int w = 1; w < others; w++)
#pragma unroll
        for (int e = 0; e < N; e++) acc[e] += sums[w][lane * N + e];
    if (VEC && live == N && tg.d_stride == 1) {
        V* p = (V*)(tg.t + (int64_t)key * tg.row_stride + c);
        V v = 0;
        if (tg.accumulate) v = *p;
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = (T)((double)v[e] + acc[e] * tg.scale);
        *p = v;
    } else {
        for (int e = 0; e < live; e++) put(tg, key, c + e, acc[e]);
    }
}

// ---- plan -----------------------------------------------------------------------------------------------------------------------------
struct GradPlan {
    uint32_t n, R, pieces, chunk, nchunks;
    int bits, npass;
    int64_t pitch;
    size_t list_bytes, counts_bytes, partial_bytes, total;
};
GradPlan grad_plan(uint32_t n, int64_t vocab, int64_t width) {
    GradPlan p;
    p.n = n;
    int kb = 1;
    while (((int64_t)1 << kb) <= vocab) kb++;   // keys are 0 .. vocab
    p.npass = (kb + kMaxDigitBits - 1) / kMaxDigitBits;
    p.bits = (kb + p.npass - 1) / p.npass;
    if (p.bits < kMinDigitBits) p.bits = kMinDigitBits;
    // pieces of 8 to 32 tokens: enough of them to fill the chip, and long enough that partials stay rare
    uint32_t R = (n + 1023) / 1024;
    R = (R + 7) / 8 * 8;
    p.R = R < 8 ? 8 : R > 32 ? 32 : R;
    p.pieces = cdiv(n, p.R);
    const uint32_t even = n / kMaxChunks + 1;
    p.chunk = (even + kSortTile - 1) / kSortTile * kSortTile;
    p.nchunks = cdiv(n, p.chunk);
    p.pitch = (width + 1) / 2 * 2;
    const bool small = n <= kSmallSort;
    if (few_tokens(n, width)) {
        p.list_bytes = p.counts_bytes = p.partial_bytes = 0;
        p.total = n ? kFewScratch : 0;
        return p;
    }
    p.list_bytes = up256((size_t)n * 4);
    p.counts_bytes = small ? 0 : up256((size_t)kMaxDigits * p.nchunks * 4);
    p.partial_bytes = up256((size_t)p.pieces * 2 * (size_t)p.pitch * 8);
    p.total = (small ? 2 : 4) * p.list_bytes + p.counts_bytes + p.partial_bytes;
    return p;
}

template <class T>
int32_t embedding_grad(const DnhTensor* dt, const DnhTensor* tokens, const DnhTensor* d_out, uint32_t n, const void* scale, int32_t accumulate, void* scratch,
                       size_t scratch_bytes, hipStream_t s) {
    const int nd = tokens->ndims;
    const int64_t vocab = dt->shape[0], width = dt->shape[1];
    ZeroRows<T> z{(T*)elem_ptr(dt), dt->stride[0], dt->stride[1], width, 0, accumulate ? 0 : vocab};
    const GradTarget<T> tg{z.t, dt->stride[0], dt->stride[1], width, (double)scalar_arg<T>(scale, 1.0), accumulate};
    const GradPlan p = grad_plan(n, vocab, width);
    TokenSource src{(const int64_t*)elem_ptr(tokens), make_row_plan<1>(nd, {tokens}), n, (uint32_t)vocab, nullptr};
    char* ws = nullptr;
    WorkspaceLease lease;
    DNH_TRY(error_flag_ptr(s, &src.err));
    const bool few = few_tokens(n, width);
    if (!few || scratch) DNH_TRY(get_scratch(s, n ? p.total : 0, scratch, scratch_bytes, (void**)&ws, lease, "dnh_embedding_grad"));
    const RowPlan<1> gp = make_row_plan<1>(nd, {d_out});
    const bool vec = d_out->stride[nd] == 1;
    if (few) {
        const unsigned chunks = cdiv(width, 64 * (vec ? kVecN<T> : 1));
        // blocks of 16 to 32 KB, a workgroup each until there are eight per compute unit
        uint32_t block_rows = 1;
        while (block_rows < kFillRows && (int64_t)block_rows * width * (int64_t)sizeof(T) < (1 << 14)) block_rows *= 2;
        const int64_t blocks = accumulate ? 0 : ((int64_t)vocab + block_rows - 1) / block_rows, most = 8 * (int64_t)device_cus();
        const unsigned grid = n * chunks + (unsigned)(blocks < most ? blocks : most);
        const int txl = lanes_log2((width + kVecN<T> - 1) / kVecN<T>);
        if (grid == 0) return DNH_OK;
        if (vec) hipLaunchKernelGGL((embedding_grad_few_kernel<T, true>), dim3(grid), dim3(kBlock), 0, s, tg, src, (const T*)elem_ptr(d_out), gp, d_out->stride[nd], chunks, block_rows, txl);
        else hipLaunchKernelGGL((embedding_grad_few_kernel<T, false>), dim3(grid), dim3(kBlock), 0, s, tg, src, (const T*)elem_ptr(d_out), gp, d_out->stride[nd], chunks, block_rows, txl);
        DNH_LAUNCH_CHECK();
        return DNH_OK;
    }
    const unsigned fill_wgs = accumulate ? 0 : (unsigned)(2 * device_cus());
    uint32_t* list[2][2];   // [buffer][keys, positions]
    for (int b = 0; b < 2; b++)
        for (int k = 0; k < 2; k++) list[b][k] = (uint32_t*)(ws + (n <= kSmallSort ? k : 2 * b + k) * p.list_bytes);
    char* rest = ws + (n <= kSmallSort ? 2 : 4) * p.list_bytes;
    uint32_t* counts = (uint32_t*)rest;
    double* partial = (double*)(rest + p.counts_bytes);
    int cur = 0;
    if (n <= kSmallSort) {
#define SORT(E) hipLaunchKernelGGL((sort_small_kernel<T, E>), dim3(1 + fill_wgs), dim3(kSortThreads), 0, s, src, p.npass, p.bits, list[0][0], list[0][1], z)
        if (n <= kSortThreads) SORT(1);
        else if (n <= 4 * kSortThreads) SORT(4);
        else SORT(8);
#undef SORT
        DNH_LAUNCH_CHECK();
    } else {
        // every launch of the sort clears a share of the target beside it: counting takes about half the time of placing
        const int parts = 3 * p.npass;
        int done = 0;
        auto share = [&](int some) {
            ZeroRows<T> part = z;
            part.row0 = z.row1 * done / parts;
            done += some;
            part.row1 = z.row1 * done / parts;
            return part;
        };
        for (int pass = 0; pass < p.npass; pass++) {
            const uint32_t* ki = pass ? list[cur][0] : nullptr;
            const uint32_t* pi = pass ? list[cur][1] : nullptr;
            hipLaunchKernelGGL((sort_count_kernel<T>), dim3(p.nchunks + fill_wgs), dim3(kSortThreads), 0, s, src, ki, pass * p.bits, p.bits, p.chunk, p.nchunks, counts, share(1));
            DNH_LAUNCH_CHECK();
            hipLaunchKernelGGL((sort_place_kernel<T>), dim3(p.nchunks + fill_wgs), dim3(kSortThreads), 0, s, src, ki, pi, pass * p.bits, p.bits, p.chunk, p.nchunks,
                               (const uint32_t*)counts, list[cur ^ 1][0], list[cur ^ 1][1], share(2));
            DNH_LAUNCH_CHECK();
            cur ^= 1;
        }
    }
    const uint32_t *keys = list[cur][0], *pos = list[cur][1];
    const int64_t items = vec ? (width + kVecN<T> - 1) / kVecN<T> : width;
    const int txl = lanes_log2(items);
    const dim3 grid(cdiv(p.pieces, kBlock >> txl), cdiv(items, (int64_t)1 << txl));
    if (vec) hipLaunchKernelGGL((embedding_sum_kernel<T, true>), grid, dim3(kBlock), 0, s, tg, (const T*)elem_ptr(d_out), gp, d_out->stride[nd], keys, pos, n, (uint32_t)vocab, txl, p.R, p.pieces, p.pitch, partial);
    else hipLaunchKernelGGL((embedding_sum_kernel<T, false>), grid, dim3(kBlock), 0, s, tg, (const T*)elem_ptr(d_out), gp, d_out->stride[nd], keys, pos, n, (uint32_t)vocab, txl, p.R, p.pieces, p.pitch, partial);
    DNH_LAUNCH_CHECK();
    if (p.pieces > 1) {
        hipLaunchKernelGGL((embedding_join_kernel<T>), dim3(p.pieces - 1, cdiv(width, kJoinCols)), dim3(kJoinThreads), 0, s, tg, keys, n, (uint32_t)vocab, p.R, p.pieces, p.pitch, (const double*)partial);
        DNH_LAUNCH_CHECK();
    }
    return DNH_OK;
}

// shapes and types both directions ask for: table [V; D], tokens [i_1 .. i_n], rows [i_1 .. i_n; D]
int32_t check_embedding(const DnhTensor* table, const DnhTensor* tokens, const DnhTensor* rows, const char* what, uint32_t* n) {
    DNH_TRY(check_float(table, table->dtype, what, "the table"));
    DNH_TRY(check_float(rows, table->dtype, what, "the tensor of rows"));
    if (tokens->dtype != DNH_I64) return fail(DNH_ERR_INVALID_ARG, "%s: tokens must be int64, not %s", what, dtype_name(tokens->dtype));
    if (table->ndims != 2) return fail(DNH_ERR_INVALID_ARG, "%s: the table must be a matrix, not of rank %d", what, table->ndims);
    if (rows->ndims != tokens->ndims + 1 || !same_leading(rows, tokens, tokens->ndims) || rows->shape[tokens->ndims] != table->shape[1])
        return fail(DNH_ERR_INVALID_ARG, "%s: the tensor of rows must have the tokens' shape followed by the table's row length %lld", what, (long long)table->shape[1]);
    if (table->shape[0] >= 0x7FFFFFFF) return fail(DNH_ERR_NOT_SUPPORTED, "%s: a table of more than 2^31 - 2 rows", what);
    if (table->shape[1] > kMaxWidth) return fail(DNH_ERR_NOT_SUPPORTED, "%s: rows of more than 2^23 elements", what);
    return count_rows(tokens, tokens->ndims, what, n);
}

}  // namespace

extern "C" int32_t dnh_embedding(const DnhTensor* t, const DnhTensor* table, const DnhTensor* tokens, const void* scale, void* stream) {
    DNH_TRY(check_target(t, "dnh_embedding", "the target"));
    DNH_TRY(check_tensor(table, "dnh_embedding"));
    DNH_TRY(check_tensor(tokens, "dnh_embedding"));
    uint32_t n;
    DNH_TRY(check_embedding(table, tokens, t, "dnh_embedding", &n));
    if (n == 0 || table->shape[1] == 0) return DNH_OK;
    DNH_TRY(check_apart<3>({t, table, tokens}, {"the target", "the table", "tokens"}, 1, "dnh_embedding"));
    DNH_TRY(ensure_init());
    hipStream_t s = (hipStream_t)stream;
    int32_t* err = nullptr;
    DNH_TRY(error_flag_ptr(s, &err));
    const bool vec = t->stride[tokens->ndims] == 1 && table->stride[1] == 1;
    if (t->dtype == DNH_F32) {
        const float sc = scalar_arg<float>(scale, 1.0);
        return vec ? launch_embedding<float, true>(t, table, tokens, n, sc, s, err) : launch_embedding<float, false>(t, table, tokens, n, sc, s, err);
    }
    const double sc = scalar_arg<double>(scale, 1.0);
    return vec ? launch_embedding<double, true>(t, table, tokens, n, sc, s, err) : launch_embedding<double, false>(t, table, tokens, n, sc, s, err);
}

extern "C" int32_t dnh_embedding_grad_scratch_bytes(int64_t tokens, int64_t vocab, int64_t width, size_t* bytes) {
    if (!bytes || tokens < 0 || vocab < 0 || width < 0 || tokens > kMaxGradTokens || vocab >= 0x7FFFFFFF || width > kMaxWidth)
        return fail(DNH_ERR_INVALID_ARG, "dnh_embedding_grad_scratch_bytes: bad argument");
    *bytes = tokens && width ? grad_plan((uint32_t)tokens, vocab, width).total : 0;
    return DNH_OK;
}

extern "C" int32_t dnh_embedding_grad(const DnhTensor* d_table, const DnhTensor* tokens, const DnhTensor* d_out, const void* scale, int32_t accumulate,
                                      void* scratch, size_t scratch_bytes, void* stream) {
    DNH_TRY(check_target(d_table, "dnh_embedding_grad", "the gradient of the table"));
    DNH_TRY(check_tensor(tokens, "dnh_embedding_grad"));
    DNH_TRY(check_tensor(d_out, "dnh_embedding_grad"));
    uint32_t n;
    DNH_TRY(check_embedding(d_table, tokens, d_out, "dnh_embedding_grad", &n));
    if (n > kMaxGradTokens) return fail(DNH_ERR_NOT_SUPPORTED, "dnh_embedding_grad: more than 2^27 tokens");
    if (accumulate != 0 && accumulate != 1) return fail(DNH_ERR_INVALID_ARG, "dnh_embedding_grad: accumulate must be 0 or 1, not %d", accumulate);
    if (d_table->shape[1] == 0 || (d_table->shape[0] == 0 && n == 0)) return DNH_OK;
    DNH_TRY(check_apart<3>({d_table, tokens, d_out}, {"the gradient of the table", "tokens", "the tensor of rows"}, 1, "dnh_embedding_grad"));
    DNH_TRY(ensure_init());
    return d_table->dtype == DNH_F32 ? embedding_grad<float>(d_table, tokens, d_out, n, scale, accumulate, scratch, scratch_bytes, (hipStream_t)stream)
                                     : embedding_grad<double>(d_table, tokens, d_out, n, scale, accumulate, scratch, scratch_bytes, (hipStream_t)stream);
}
