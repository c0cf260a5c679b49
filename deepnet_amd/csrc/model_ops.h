// Shared by the language-model operators (embedding.hip, logprobs.hip, attention.hip): row addressing, 16-byte vectors at element
// alignment, scalar arguments and the choice between the caller's scratch memory and the stream's workspace.
#pragma once

#include "common.h"

#include <type_traits>

namespace dnh {

// 16 bytes of T at T's own alignment (the hardware serves 16-byte accesses at any dword address, so views that start at an odd
// element or have odd pitches keep the wide accesses)
template <class T> struct Vec16;
template <> struct Vec16<float> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Vec16<double> { typedef double type __attribute__((ext_vector_type(2), aligned(8))); };
template <class T> constexpr int kVecN = 16 / (int)sizeof(T);

// The leading dimensions [i_1 .. i_n] that K operands share, in row-major order of the rows: extent-1 dimensions dropped, neighbours
// that chain for every operand merged, so that contiguous operands are addressed without a division.
template <int K> struct RowPlan {
    int nd;
    uint32_t shape[DNH_MAX_DIMS];
    int64_t stride[K][DNH_MAX_DIMS];
};

template <int K> RowPlan<K> make_row_plan(int ndims, const DnhTensor* const (&ops)[K]) {
    RowPlan<K> p;
    memset(&p, 0, sizeof(p));
    for (int d = 0; d < ndims; d++) {
        const int64_t n = ops[0]->shape[d];
        if (n == 1) continue;
        bool chain = p.nd > 0;
        for (int k = 0; k < K && chain; k++) chain = p.stride[k][p.nd - 1] == ops[k]->stride[d] * n;
        if (chain) {
            p.shape[p.nd - 1] *= (uint32_t)n;
        } else {
            p.shape[p.nd] = (uint32_t)n;
            p.nd++;
        }
        for (int k = 0; k < K; k++) p.stride[k][p.nd - 1] = ops[k]->stride[d];
    }
    return p;
}

template <int K> __device__ __forceinline__ void row_offsets(const RowPlan<K>& p, uint32_t i, int64_t (&off)[K]) {
#pragma unroll
    for (int k = 0; k < K; k++) off[k] = 0;
    for (int d = p.nd - 1; d >= 0; d--) {
        const uint32_t q = d == 0 ? 0u : i / p.shape[d];
        const int64_t pos = i - q * p.shape[d];
#pragma unroll
        for (int k = 0; k < K; k++) off[k] += pos * p.stride[k][d];
        i = q;
    }
}

// rows of the leading `ndims` dimensions; more than 2^31 - 1 are refused
inline int32_t count_rows(const DnhTensor* t, int ndims, const char* what, uint32_t* rows) {
    int64_t n = 1;
    for (int d = 0; d < ndims; d++) n *= t->shape[d];
    if (n > 0x7FFFFFFF) return fail(DNH_ERR_NOT_SUPPORTED, "%s: more than 2^31 - 1 rows", what);
    *rows = (uint32_t)n;
    return DNH_OK;
}

inline bool same_leading(const DnhTensor* a, const DnhTensor* b, int ndims) {
    for (int d = 0; d < ndims; d++)
        if (a->shape[d] != b->shape[d]) return false;
    return true;
}

// A target whose elements share memory (a broadcast view) would be written by several threads.
inline int32_t check_target(const DnhTensor* t, const char* what, const char* name) {
    DNH_TRY(check_tensor(t, what));
    if (nelems(t) == 0) return DNH_OK;
    for (int d = 0; d < t->ndims; d++)
        if (t->shape[d] > 1 && t->stride[d] == 0) return fail(DNH_ERR_INVALID_ARG, "%s: %s is a broadcast view", what, name);
    return DNH_OK;
}

// ---- targets that share memory with a source or with each other ------------------------------------------------------------------
// Whether two views certainly have a byte in common: both fill the ranges they span, and those meet; or a corner of one (its first or last
// position along every axis) is an element of the other.  Views that interleave (heads beside each other in one tensor) do not count.
struct Span {
    int64_t lo = 0, hi = 0;   // addresses of the first and behind the last byte
    int nd = 0;               // axes of more than one position, by descending stride, all positive
    int64_t n[DNH_MAX_DIMS], stride[DNH_MAX_DIMS];
    bool nested = true;       // every stride is longer than what the axes behind it reach: positions and addresses are one to one
    int esize = 0;
};
inline Span span_of(const DnhTensor* t) {
    Span s;
    s.esize = dtype_size(t->dtype);
    s.lo = (int64_t)(intptr_t)t->base + t->offset * s.esize;
    int64_t last = 0;
    for (int d = 0; d < t->ndims; d++) {
        if (t->shape[d] < 2 || t->stride[d] == 0) continue;
        const int64_t st = (t->stride[d] < 0 ? -t->stride[d] : t->stride[d]) * s.esize, reach = st * (t->shape[d] - 1);
        if (t->stride[d] < 0) s.lo -= reach;
        last += reach;
        int at = s.nd++;
        for (; at > 0 && s.stride[at - 1] < st; at--) {
            s.stride[at] = s.stride[at - 1];
            s.n[at] = s.n[at - 1];
        }
        s.stride[at] = st;
        s.n[at] = t->shape[d];
    }
    s.hi = s.lo + last + s.esize;
    int64_t inner = s.esize;
    for (int d = s.nd - 1; d >= 0; d--) {
        if (s.stride[d] < inner) s.nested = false;
        inner += s.stride[d] * (s.n[d] - 1);
    }
    return s;
}
inline bool fills(const Span& s) {
    int64_t bytes = s.esize;
    for (int d = 0; d < s.nd; d++) bytes *= s.n[d];
    return s.nested && bytes == s.hi - s.lo;
}
inline bool has_corner_of(const Span& a, const Span& b) {   // equal element sizes
    if (!a.nested) return false;
    for (int c = 0; c < 1 << b.nd; c++) {
        int64_t at = b.lo - a.lo;
        for (int d = 0; d < b.nd; d++)
            if ((c >> d) & 1) at += b.stride[d] * (b.n[d] - 1);
        bool in = at >= 0;
        for (int d = 0; d < a.nd && in; d++) {
            const int64_t i = at / a.stride[d];
            in = i < a.n[d];
            at -= i * a.stride[d];
        }
        if (in && at == 0) return true;
    }
    return false;
}
inline bool surely_overlap(const Span& a, const Span& b) {
    if (a.hi <= b.lo || b.hi <= a.lo) return false;
    if (fills(a) && fills(b)) return true;
    return a.esize == b.esize && (has_corner_of(a, b) || has_corner_of(b, a));
}
inline bool same_view(const DnhTensor* x, const DnhTensor* y) {
    if (x->base != y->base || x->offset != y->offset || x->ndims != y->ndims || x->dtype != y->dtype) return false;
    for (int d = 0; d < x->ndims; d++)
        if (x->shape[d] != y->shape[d] || (x->shape[d] > 1 && x->stride[d] != y->stride[d])) return false;
    return true;
}
// targets before sources; any may be NULL
template <int N> int32_t check_apart(const DnhTensor* const (&ts)[N], const char* const (&names)[N], int targets, const char* what) {
    Span s[N];
    for (int i = 0; i < N; i++)
        if (ts[i] && nelems(ts[i]) > 0) s[i] = span_of(ts[i]);   // (else an empty range, which meets none)
    for (int i = 0; i < targets; i++)
        for (int j = i + 1; j < N; j++)
            if (surely_overlap(s[i], s[j])) return fail(DNH_ERR_INVALID_ARG, "%s: %s overlaps %s in memory", what, names[i], names[j]);
    return DNH_OK;
}

inline int32_t check_float(const DnhTensor* t, int32_t dtype, const char* what, const char* name) {
    if (!dtype_is_fp(t->dtype)) return fail(DNH_ERR_NOT_SUPPORTED, "%s on %s", what, dtype_name(t->dtype));
    if (t->dtype != dtype) return fail(DNH_ERR_INVALID_ARG, "%s: %s is %s, not %s", what, name, dtype_name(t->dtype), dtype_name(dtype));
    return DNH_OK;
}

// One host element of the operands' type, or the default where the caller passes NULL.
template <class T> T scalar_arg(const void* value, double dflt) {
    if (!value) return (T)dflt;
    T v;
    memcpy(&v, value, sizeof(v));
    return v;
}

// Memory for a call's intermediates: the caller's, or the stream's workspace.  A call that is being captured into a graph takes the
// caller's only: the workspace may move when a later call needs more of it, and is shared by everything on the stream, while a
// graph keeps the addresses it was captured with and may be replayed beside another.
inline int32_t get_scratch(hipStream_t stream, size_t need, void* given, size_t given_bytes, void** out, WorkspaceLease& lease, const char* what) {
    *out = nullptr;
    if (need == 0) return DNH_OK;
    if (given) {
        if (given_bytes < need) return fail(DNH_ERR_INVALID_ARG, "%s: %zu bytes of scratch memory, %zu needed", what, given_bytes, need);
        if ((uintptr_t)given % 16 != 0) return fail(DNH_ERR_INVALID_ARG, "%s: scratch memory must be aligned to 16 bytes", what);
        *out = given;
        return DNH_OK;
    }
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    DNH_HIP(hipStreamIsCapturing(stream, &st));
    if (st != hipStreamCaptureStatusNone)
        return fail(DNH_ERR_INVALID_ARG, "%s: a call that is captured into a graph needs scratch memory of its own (%zu bytes)", what, need);
    return workspace(stream, need, out, lease);
}

// Between LDS accesses of one wavefront whose lanes hand each other data: the hardware serves them in order, and this keeps the compiler from
// moving them across or from using again what a lane has read before.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

inline size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// Threads of a 256-thread workgroup that share a row of `items` accesses: a power of two of 4..256.
inline int lanes_log2(int64_t items) {
    int l = 2;
    while (l < 8 && ((int64_t)1 << l) < items) l++;
    return l;
}

constexpr int64_t kMaxWidth = (int64_t)1 << 23;   // elements of a row that is spread over a grid's second dimension

}  // namespace dnh
