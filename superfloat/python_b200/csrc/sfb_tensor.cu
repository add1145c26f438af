// Entry points of the tensor-core linear: checks, and the launches in order.  One
// call queues a whole pass, so that a caller pays for one crossing of the boundary.
#include "sfb_tensor_parts.cuh"

namespace sfb {
namespace {

bool is_16(int64_t t) { return t == SFB_BF16 || t == SFB_F16; }
bool is_float(int64_t t) { return t == SFB_F32 || is_16(t); }
bool on16(const void *p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }

int check(const sfb_tensor_call *c, const char *what, bool codes) {
    if (!c) return set_error(SFB_EINVAL, "%s: null pointer", what);
    if (!is_16(c->dtype)) return set_error(SFB_EINVAL, "%s: element type %d", what, (int)c->dtype);
    if (c->bits < 4 || c->bits > 8) return set_error(SFB_EINVAL, "%s: width %d is not in 4..8", what, (int)c->bits);
    if (c->act < SFB_ACT_NONE || c->act > SFB_ACT_SILU)
        return set_error(SFB_EINVAL, "%s: activation %d", what, (int)c->act);
    if (c->M < 0 || c->N < 1 || c->K < 1) return set_error(SFB_EINVAL, "%s: bad shape", what);
    // tile coordinates are 32-bit
    if (c->M >= (1ll << 31) - 512 || c->N >= (1ll << 31) - 512 || c->K >= (1ll << 31) - 512 ||
        ((c->N + 255) / 256) * ((c->M + 127) / 128) >= (1ll << 31) || ((c->K + 255) / 256) * ((c->M + 127) / 128) >= (1ll << 31) ||
        ((c->K + 255) / 256) * ((c->N + 127) / 128) >= (1ll << 31))
        return set_error(SFB_ERANGE, "%s: a size of %lld x %lld x %lld", what, (long long)c->M, (long long)c->N,
                         (long long)c->K);
    if (codes && (!c->codes || !on16(c->codes, c->ldc) || c->ldc < c->K))
        return set_error(SFB_EINVAL, "%s: the codes' rows must start on 16 bytes", what);
    if (!c->scale) return set_error(SFB_EINVAL, "%s: null pointer", what);
    return SFB_OK;
}

}  // namespace
}  // namespace sfb

extern "C" int sfb_tensor_forward(const sfb_tensor_call *c, sfb_stream stream) {
    using namespace sfb;
    const char *what = "sfb_tensor_forward";
    if (!c) return set_error(SFB_EINVAL, "%s: null pointer", what);
    const bool packed = c->w_dtype == SFB_I8, small = packed && c->codes == nullptr;
    int rc = check(c, what, !small);
    if (rc) return rc;
    if (small && (c->M > SFB_SMALL_ROWS || c->z))
        return set_error(SFB_EINVAL, "%s: more than %d rows, or a pre-activation to keep, and no room for the codes",
                         what, SFB_SMALL_ROWS);
    if (!packed && !is_float(c->w_dtype)) return set_error(SFB_EINVAL, "%s: weight type %d", what, (int)c->w_dtype);
    if (c->ldx < c->K || c->ldw < c->K || c->ldy < c->N || (c->residual && c->ldr < c->N) || (c->z && c->ldz < c->N))
        return set_error(SFB_EINVAL, "%s: a row stride is shorter than its row", what);
    if (c->bias && !is_float(c->bias_dtype)) return set_error(SFB_EINVAL, "%s: bias type %d", what, (int)c->bias_dtype);
    if (!c->w || (!packed && !c->per_channel && !c->work)) return set_error(SFB_EINVAL, "%s: null pointer", what);
    if (c->M > 0 && (!c->x || !c->y)) return set_error(SFB_EINVAL, "%s: null pointer", what);
    const bool pad = c->M > 0 && !on16(c->x, c->ldx);
    if (pad && (!c->xpad || !on16(c->xpad, c->ldp) || c->ldp < c->K))
        return set_error(SFB_EINVAL, "%s: x does not start on 16 bytes and there is no room for a copy", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    float *scale = const_cast<float *>(c->scale);
    const int t = (int)c->dtype, bits = (int)c->bits, bd = (int)c->bias_dtype, act = (int)c->act;
    const Rows rows{pad ? c->x : nullptr, c->M, c->K, c->ldx, c->xpad, c->ldp};
    if (!packed)
        rc = tensor_quantize(c->w, (int)c->w_dtype, c->N, c->K, c->ldw, bits, c->per_channel != 0, c->codes, c->ldc, t,
                             scale, c->work, rows, st);
    else if (!small && c->M > 0)
        rc = tensor_expand(static_cast<const int8_t *>(c->w), c->N, c->K, c->ldw, c->codes, c->ldc, t, rows, st);
    else if (pad)
        rc = tensor_pad(rows, st);
    if (rc || c->M == 0) return rc;
    const void *x = pad ? c->xpad : c->x;
    const int64_t ldx = pad ? c->ldp : c->ldx;
    if (small)
        return tensor_small(t, x, ldx, static_cast<const int8_t *>(c->w), c->ldw, scale, bits, c->bias, bd, act,
                            c->residual, c->ldr, c->y, c->ldy, c->M, c->N, c->K, st);
    return tensor_product(t, x, ldx, c->codes, c->ldc, scale, bits, c->bias, bd, act, c->residual, c->ldr, c->y, c->ldy,
                          c->z, c->ldz, c->M, c->N, c->K, st);
}

extern "C" int64_t sfb_tensor_sums(int64_t M, int64_t N) { return 4 * sfb::tensor_slope_parts(M) * N; }

extern "C" int sfb_tensor_backward(const sfb_tensor_call *c, sfb_stream stream) {
    using namespace sfb;
    const char *what = "sfb_tensor_backward";
    int rc = check(c, what, true);
    if (rc) return rc;
    if (c->M == 0) return set_error(SFB_EINVAL, "%s: no rows", what);
    if (c->ldx < c->K || c->ldy < c->N || (c->act != SFB_ACT_NONE && c->ldz < c->N) || c->ldd < c->N || c->ldd % 8)
        return set_error(SFB_EINVAL, "%s: a row stride is shorter than its row", what);
    if (!c->x || !c->y || (c->act != SFB_ACT_NONE && !c->z)) return set_error(SFB_EINVAL, "%s: null pointer", what);
    if (!on16(c->x, c->ldx)) return set_error(SFB_EINVAL, "%s: x does not start on 16 bytes", what);
    if ((c->db && (!is_float(c->db_dtype) || !c->work)) || (c->dw && !is_float(c->w_dtype)))
        return set_error(SFB_EINVAL, "%s: a gradient's type", what);
    // One scale: dz s / top is dz, an operand of both products.  Without an activation, and where its rows start on 16
    // bytes, that is the result's gradient as it came.
    const bool one = c->per_channel == 0, direct = c->act == SFB_ACT_NONE && on16(c->y, c->ldy);
    const bool need_dz = (c->dw || (c->dx && one)) && !direct, need_dzs = c->dx && !one;
    if ((need_dz && (!c->dz || !on16(c->dz, 0))) || (need_dzs && (!c->dzs || !on16(c->dzs, 0))))
        return set_error(SFB_EINVAL, "%s: no room for the pre-activation's gradient", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int t = (int)c->dtype, bits = (int)c->bits;
    // fp16: dz s would leave its range where the scales are small; s over the largest one with a code is within it
    const float *top = one ? c->scale : nullptr;
    if (need_dzs && t == SFB_F16) {
        if (!c->top) return set_error(SFB_EINVAL, "%s: null pointer", what);
        top = c->top;
        rc = tensor_top(c->scale, c->N, c->codes, c->ldc, c->K, c->top, st);
        if (rc) return rc;
    }
    float *parts = c->db ? static_cast<float *>(c->work) : nullptr;
    if (need_dz || need_dzs || c->db)
        rc = tensor_slope(t, (int)c->act, c->y, c->ldy, c->z, c->ldz, c->M, c->N, c->scale, bits, top,
                          need_dz ? c->dz : nullptr, need_dzs ? c->dzs : nullptr, c->ldd, parts, st);
    if (rc) return rc;
    const Sums sums{parts, tensor_slope_parts(c->M), c->N, c->db, (int)c->db_dtype};
    const void *dz = direct ? c->y : c->dz;
    const int64_t ldd = direct ? c->ldy : c->ldd;
    if (c->dx)
        rc = tensor_grad_x(t, one ? dz : c->dzs, one ? ldd : c->ldd, c->codes, c->ldc, top, bits, c->dx, c->K, c->M,
                           c->N, c->K, st);
    if (rc) return rc;
    if (c->dw)
        rc = tensor_grad_w(t, dz, ldd, c->x, c->ldx, c->dw, (int)c->w_dtype, c->K, c->M, c->N, c->K, sums, st);
    else if (parts)
        rc = tensor_sum(sums, st);
    return rc;
}
