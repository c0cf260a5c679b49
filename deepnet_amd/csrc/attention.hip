// dnh_cross_attention, dnh_cross_attention_grad: attention of queries to an encoder's states of another length, and its gradient.
// The kernels and their mathematics are in attention_kernels.h.
#include "attention_kernels.h"

namespace dnh {
template <> int32_t attention_forward<float>(AttArgs<float>& p, void* scratch, size_t scratch_bytes, hipStream_t s) { return attention_forward_impl<float>(p, scratch, scratch_bytes, s); }
template <> int32_t attention_backward<float>(AttArgs<float>& p, void* scratch, size_t scratch_bytes, hipStream_t s) { return attention_backward_impl<float>(p, scratch, scratch_bytes, s); }
}  // namespace dnh

using namespace dnh;

namespace {

constexpr int64_t kMaxHeadWidth = 128;

Strides4 strides4(const DnhTensor* t) { return Strides4{t->stride[0], t->stride[1], t->stride[2], t->ndims > 3 ? t->stride[3] : 0}; }

// 32-bit counts inside the kernels (extents, rows of a key head, heads), and grids of fewer than 2^32 threads: at most 2^23 tiles of 64 rows,
// as many of 64 keys, and 2^28 rows for the kernels that give each 16 lanes or more
int32_t check_extents(int64_t batch, int64_t heads, int64_t kv_heads, int64_t queries, int64_t keys, const char* what) {
    const int64_t lim = 0x7FFFFFFF - 16384;
    if (batch > lim || heads > lim || kv_heads > lim || queries > lim || keys > lim) return fail(DNH_ERR_NOT_SUPPORTED, "%s: an extent of 2^31 or more", what);
    if (kv_heads == 0) return DNH_OK;
    const int64_t rows = heads / kv_heads * queries, n = batch * kv_heads;
    if (n > (1 << 23) || rows > lim || n * (rows / 32 + 1) >= (1 << 23) || n * (keys / 64 + 1) >= (1 << 23))
        return fail(DNH_ERR_NOT_SUPPORTED, "%s: more than 2^23 tiles of rows or keys", what);
    return DNH_OK;
}

// The operands both directions share: q [B; Hq; Lq; Dk], k [B; Hk; Lk; Dk], v [B; Hk; Lk; Dv], mask [B; Lk] or NULL
int32_t check_operands(const DnhTensor* q, const DnhTensor* k, const DnhTensor* v, const DnhTensor* mask, const char* what) {
    const DnhTensor* ts[] = {q, k, v};
    const char* names[] = {"q", "k", "v"};
    for (int i = 0; i < 3; i++) {
        DNH_TRY(check_tensor(ts[i], what));
        DNH_TRY(check_float(ts[i], q->dtype, what, names[i]));
        if (ts[i]->ndims != 4) return fail(DNH_ERR_INVALID_ARG, "%s: %s must have the axes [batch; head; position; width], but is of rank %d", what, names[i], ts[i]->ndims);
    }
    if (k->shape[0] != q->shape[0] || v->shape[0] != q->shape[0]) return fail(DNH_ERR_INVALID_ARG, "%s: q, k and v must have the same batch extent", what);
    if (k->shape[1] != v->shape[1] || k->shape[2] != v->shape[2]) return fail(DNH_ERR_INVALID_ARG, "%s: k and v must have the same heads and positions", what);
    if (k->shape[3] != q->shape[3]) return fail(DNH_ERR_INVALID_ARG, "%s: q and k must have the same width, but have %lld and %lld", what, (long long)q->shape[3], (long long)k->shape[3]);
    if (k->shape[1] == 0 ? q->shape[1] != 0 : q->shape[1] % k->shape[1] != 0)
        return fail(DNH_ERR_INVALID_ARG, "%s: %lld query heads cannot share %lld key heads evenly", what, (long long)q->shape[1], (long long)k->shape[1]);
    if (q->shape[3] < 1 || v->shape[3] < 1) return fail(DNH_ERR_INVALID_ARG, "%s: heads without a width", what);
    if (q->shape[3] > kMaxHeadWidth || v->shape[3] > kMaxHeadWidth) return fail(DNH_ERR_NOT_SUPPORTED, "%s: heads wider than %lld", what, (long long)kMaxHeadWidth);
    if (mask) {
        DNH_TRY(check_tensor(mask, what));
        if (mask->dtype != DNH_BOOL || mask->ndims != 2 || mask->shape[0] != k->shape[0] || mask->shape[1] != k->shape[2])
            return fail(DNH_ERR_INVALID_ARG, "%s: the mask must be a bool tensor [batch; key position]", what);
    }
    return check_extents(q->shape[0], q->shape[1], k->shape[1], q->shape[2], k->shape[2], what);
}

int32_t check_like(const DnhTensor* t, const DnhTensor* q, int64_t heads, int64_t len, int64_t width, const char* what, const char* name, bool target) {
    DNH_TRY(target ? check_target(t, what, name) : check_tensor(t, what));
    if (t->dtype != q->dtype || t->ndims != 4 || t->shape[0] != q->shape[0] || t->shape[1] != heads || t->shape[2] != len || t->shape[3] != width)
        return fail(DNH_ERR_INVALID_ARG, "%s: %s must be a %s tensor [%lld; %lld; %lld; %lld]", what, name, dtype_name(q->dtype), (long long)q->shape[0], (long long)heads,
                    (long long)len, (long long)width);
    return DNH_OK;
}
int32_t check_lse(const DnhTensor* t, const DnhTensor* q, const char* what, bool target) {
    DNH_TRY(target ? check_target(t, what, "lse") : check_tensor(t, what));
    if (t->dtype != q->dtype || t->ndims != 3 || !same_leading(t, q, 3)) return fail(DNH_ERR_INVALID_ARG, "%s: lse must be a %s tensor [batch; head; position] of q", what, dtype_name(q->dtype));
    return DNH_OK;
}

template <class T>
AttArgs<T> common_args(const DnhTensor* q, const DnhTensor* k, const DnhTensor* v, const DnhTensor* mask, const void* scale) {
    AttArgs<T> p;
    memset((void*)&p, 0, sizeof(p));
    p.q = (const T*)elem_ptr(q);
    p.k = (const T*)elem_ptr(k);
    p.v = (const T*)elem_ptr(v);
    p.sq = strides4(q);
    p.sk = strides4(k);
    p.sv = strides4(v);
    if (mask) {
        p.mask = (const uint8_t*)elem_ptr(mask);
        p.mask_b = mask->stride[0];
        p.mask_l = mask->stride[1];
    }
    p.B = (int)q->shape[0];
    p.Hk = (int)k->shape[1];
    p.G = p.Hk ? (int)(q->shape[1] / k->shape[1]) : 0;
    p.Lq = (int)q->shape[2];
    p.Lk = (int)k->shape[2];
    p.Dk = (int)q->shape[3];
    p.Dv = (int)v->shape[3];
    p.rows = (uint32_t)p.G * (uint32_t)p.Lq;
    p.scale = scalar_arg<T>(scale, 1.0 / sqrt((double)p.Dk));
    p.scale_base = (T)((double)p.scale * MmaOf<T>::Tile::kBase);
    p.vec = p.sq.d == 1 && p.sk.d == 1 && p.sv.d == 1;
    p.whole = p.vec && p.Dk % kVecN<T> == 0 && p.Dv % kVecN<T> == 0;
    p.exact = option(OPT_ATTENTION_BF16X3) == 0;
    // with 2^(l - 1) < Lq <= 2^l and mul = ceil(2^(31 + l) / Lq): mul Lq exceeds 2^(31 + l) by less than 2^l, so r mul 2^-(31 + l) exceeds
    // r / Lq by less than r 2^-31 / Lq < 1 / Lq, and the integer parts agree
    int l = 0;
    while (((int64_t)1 << l) < p.Lq) l++;
    p.lq_shift = 31 + l;
    p.lq_mul = p.Lq > 0 ? (uint32_t)((((uint64_t)1 << (31 + l)) + p.Lq - 1) / p.Lq) : 0;
    return p;
}

template <class T>
int32_t forward(const DnhTensor* out, const DnhTensor* lse, const DnhTensor* q, const DnhTensor* k, const DnhTensor* v, const DnhTensor* mask, const void* scale,
                void* scratch, size_t scratch_bytes, hipStream_t s) {
    AttArgs<T> p = common_args<T>(q, k, v, mask, scale);
    p.o = (T*)elem_ptr(out);
    p.so = strides4(out);
    if (lse) {
        p.lse_out = (T*)elem_ptr(lse);
        p.slse = strides4(lse);
    }
    return attention_forward<T>(p, scratch, scratch_bytes, s);
}

template <class T>
int32_t backward(const DnhTensor* dq, const DnhTensor* dk, const DnhTensor* dv, const DnhTensor* d_out, const DnhTensor* q, const DnhTensor* k, const DnhTensor* v,
                 const DnhTensor* out, const DnhTensor* lse, const DnhTensor* mask, const void* scale, void* scratch, size_t scratch_bytes, hipStream_t s) {
    AttArgs<T> p = common_args<T>(q, k, v, mask, scale);
    p.out = (const T*)elem_ptr(out);
    p.so = strides4(out);
    p.d_out = (const T*)elem_ptr(d_out);
    p.sdo = strides4(d_out);
    p.lse = (const T*)elem_ptr(lse);
    p.slse = strides4(lse);
    p.vec = p.vec && p.sdo.d == 1;
    p.whole = p.whole && p.vec;
    if (dq) {
        p.dq = (T*)elem_ptr(dq);
        p.sdq = strides4(dq);
    }
    if (dk) {
        p.dk = (T*)elem_ptr(dk);
        p.sdk = strides4(dk);
        p.dv = (T*)elem_ptr(dv);
        p.sdv = strides4(dv);
    }
    return attention_backward<T>(p, scratch, scratch_bytes, s);
}

}  // namespace

extern "C" int32_t dnh_cross_attention_scratch_bytes(int32_t dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t queries, int64_t keys, int64_t width,
                                                     size_t* bytes) {
    if (!bytes || !dtype_is_fp(dtype) || batch < 0 || kv_heads < 1 || heads < 0 || heads % kv_heads != 0 || queries < 0 || keys < 0 || width < 1 || width > kMaxHeadWidth)
        return fail(DNH_ERR_INVALID_ARG, "dnh_cross_attention_scratch_bytes: bad argument");
    DNH_TRY(check_extents(batch, heads, kv_heads, queries, keys, "dnh_cross_attention_scratch_bytes"));
    const int64_t n = batch * kv_heads, rows = heads / kv_heads * queries;
    *bytes = 0;
    if (n == 0 || rows == 0) return DNH_OK;
    const size_t f = dtype == DNH_F32 ? att_plan<float>(n, rows, keys, width, width).total : att_plan<double>(n, rows, keys, width, width).total;
    const size_t b = dtype == DNH_F32 ? att_grad_plan<float>(n, rows, keys, width, width).total : att_grad_plan<double>(n, rows, keys, width, width).total;
    *bytes = f > b ? f : b;
    return DNH_OK;
}

extern "C" int32_t dnh_cross_attention(const DnhTensor* out, const DnhTensor* lse, const DnhTensor* q, const DnhTensor* k, const DnhTensor* v, const DnhTensor* mask,
                                       const void* scale, void* scratch, size_t scratch_bytes, void* stream) {
    const char* what = "dnh_cross_attention";
    DNH_TRY(check_operands(q, k, v, mask, what));
    DNH_TRY(check_like(out, q, q->shape[1], q->shape[2], v->shape[3], what, "out", true));
    if (lse) DNH_TRY(check_lse(lse, q, what, true));
    if (nelems(out) == 0) return DNH_OK;
    DNH_TRY(check_apart<6>({out, lse, q, k, v, mask}, {"out", "lse", "q", "k", "v", "the mask"}, 2, what));
    DNH_TRY(ensure_init());
    return q->dtype == DNH_F32 ? forward<float>(out, lse, q, k, v, mask, scale, scratch, scratch_bytes, (hipStream_t)stream)
                               : forward<double>(out, lse, q, k, v, mask, scale, scratch, scratch_bytes, (hipStream_t)stream);
}

extern "C" int32_t dnh_cross_attention_grad(const DnhTensor* d_q, const DnhTensor* d_k, const DnhTensor* d_v, const DnhTensor* d_out, const DnhTensor* q, const DnhTensor* k,
                                            const DnhTensor* v, const DnhTensor* out, const DnhTensor* lse, const DnhTensor* mask, const void* scale, void* scratch,
                                            size_t scratch_bytes, void* stream) {
    const char* what = "dnh_cross_attention_grad";
    DNH_TRY(check_operands(q, k, v, mask, what));
    if (!d_k != !d_v) return fail(DNH_ERR_INVALID_ARG, "%s: d_k and d_v are given together or not at all", what);
    if (!d_q && !d_k) return fail(DNH_ERR_INVALID_ARG, "%s: nothing to compute", what);
    DNH_TRY(check_like(d_out, q, q->shape[1], q->shape[2], v->shape[3], what, "d_out", false));
    DNH_TRY(check_like(out, q, q->shape[1], q->shape[2], v->shape[3], what, "out", false));
    DNH_TRY(check_lse(lse, q, what, false));
    if (d_q) DNH_TRY(check_like(d_q, q, q->shape[1], q->shape[2], q->shape[3], what, "d_q", true));
    if (d_k) {
        DNH_TRY(check_like(d_k, q, k->shape[1], k->shape[2], k->shape[3], what, "d_k", true));
        DNH_TRY(check_like(d_v, q, v->shape[1], v->shape[2], v->shape[3], what, "d_v", true));
    }
    if ((!d_q || nelems(d_q) == 0) && (!d_k || nelems(d_k) == 0)) return DNH_OK;
    DNH_TRY(check_apart<10>({d_q, d_k, d_v, d_out, q, k, v, out, lse, mask}, {"d_q", "d_k", "d_v", "d_out", "q", "k", "v", "out", "lse", "the mask"}, 3, what));
    DNH_TRY(ensure_init());
    return q->dtype == DNH_F32 ? backward<float>(d_q, d_k, d_v, d_out, q, k, v, out, lse, mask, scale, scratch, scratch_bytes, (hipStream_t)stream)
                               : backward<double>(d_q, d_k, d_v, d_out, q, k, v, out, lse, mask, scale, scratch, scratch_bytes, (hipStream_t)stream);
}
