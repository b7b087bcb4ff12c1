// C entry points of the operators over packed rows (include/mfcc_hip.h): argument checks, then the launches
// of packed_conv.h / packed_scan.h / packed_norm.h for the element type (packed_inst.hip).
#include "packed_conv.h"
#include "packed_norm.h"
#include "packed_scan.h"

using mfcc_detail::fail;

namespace packed {
#define DECLARE_TYPE(T)                                                                     \
    extern template int conv_forward<T>(const mfcc_conv_args*, hipStream_t);                \
    extern template int conv_backward<T>(const mfcc_conv_args*, hipStream_t);               \
    extern template int conv_step<T>(ConvStep, int, hipStream_t);                           \
    extern template int scan_forward<T>(const mfcc_scan_args*, hipStream_t);                \
    extern template int scan_backward<T>(const mfcc_scan_args*, hipStream_t);               \
    extern template int scan_step<T>(const mfcc_scan_args*, int, const int32_t*, hipStream_t); \
    extern template int add_norm_forward<T>(const mfcc_norm_args*, hipStream_t);            \
    extern template int add_norm_backward<T>(const mfcc_norm_args*, hipStream_t);           \
    extern template int gate_norm_forward<T>(const mfcc_norm_args*, hipStream_t);           \
    extern template int gate_norm_backward<T>(const mfcc_norm_args*, hipStream_t);
DECLARE_TYPE(F32)
DECLARE_TYPE(BF16)
DECLARE_TYPE(F16)
}  // namespace packed

using namespace packed;

namespace {

constexpr int MAX_CHANNELS = 1 << 24;

int check_conv(const mfcc_conv_args* a) {
    if (!a || a->struct_size != (int32_t)sizeof(mfcc_conv_args)) return fail(MFCC_E_INVALID, "mfcc_conv_args of another size");
    if (a->dtype < MFCC_F32 || a->dtype > MFCC_F16) return fail(MFCC_E_INVALID, "unknown element type");
    if (a->rows < 0 || a->channels < 1 || a->channels > MAX_CHANNELS || a->n_seqs < 0)
        return fail(MFCC_E_INVALID, "bad convolution shape");
    if (a->width < 1 || a->width > 8) return fail(MFCC_E_INVALID, "width must lie between 1 and 8");
    if (a->activation != MFCC_ACT_NONE && a->activation != MFCC_ACT_SILU) return fail(MFCC_E_INVALID, "unknown activation");
    if (!a->d_offsets && a->n_seqs != 1) return fail(MFCC_E_INVALID, "n_seqs must be 1 without offsets");
    if (a->rows > 0 && a->n_seqs == 0) return fail(MFCC_E_INVALID, "rows without a sequence");
    if (!a->d_weight) return fail(MFCC_E_INVALID, "NULL weight");
    return MFCC_OK;
}

int check_scan(const mfcc_scan_args* a, bool step) {
    if (!a || a->struct_size != (int32_t)sizeof(mfcc_scan_args)) return fail(MFCC_E_INVALID, "mfcc_scan_args of another size");
    if (a->dtype < MFCC_F32 || a->dtype > MFCC_F16) return fail(MFCC_E_INVALID, "unknown element type");
    if (a->rows < 0 || a->channels < 1 || a->channels > MAX_CHANNELS || a->n_seqs < 0) return fail(MFCC_E_INVALID, "bad scan shape");
    if (a->state < 1) return fail(MFCC_E_INVALID, "state must be positive");
    if (a->state > 64) return fail(MFCC_E_UNSUPPORTED, "more than 64 states per channel");
    if (a->groups < 1 || a->channels % a->groups) return fail(MFCC_E_INVALID, "channels must be a multiple of groups");
    if (!step && !a->d_offsets && a->n_seqs != 1) return fail(MFCC_E_INVALID, "n_seqs must be 1 without offsets");
    if (!step && a->rows > 0 && a->n_seqs == 0) return fail(MFCC_E_INVALID, "rows without a sequence");
    if (!a->d_A) return fail(MFCC_E_INVALID, "NULL A");
    if (a->rows > 0 && (!a->d_u || !a->d_delta || !a->d_B || !a->d_C)) return fail(MFCC_E_INVALID, "NULL scan buffer");
    return MFCC_OK;
}

int check_norm(const mfcc_norm_args* a, bool gate) {
    if (!a || a->struct_size != (int32_t)sizeof(mfcc_norm_args)) return fail(MFCC_E_INVALID, "mfcc_norm_args of another size");
    if (a->dtype < MFCC_F32 || a->dtype > MFCC_F16) return fail(MFCC_E_INVALID, "unknown element type");
    if (a->rows < 0 || a->channels < 1 || a->groups < 1 || a->groups > 65535 || a->channels % a->groups)
        return fail(MFCC_E_INVALID, "bad norm shape");
    if (!gate && (a->groups != 1 || (a->res_dtype != a->dtype && a->res_dtype != MFCC_F32)))
        return fail(MFCC_E_INVALID, "the residual is of the element type or float32, in one group");
    if (a->channels / a->groups > NORM_MAX_WIDTH) return fail(MFCC_E_UNSUPPORTED, "rows wider than 32768");
    if (a->norm != MFCC_NORM_RMS && a->norm != MFCC_NORM_LAYER) return fail(MFCC_E_INVALID, "unknown norm");
    if (!(a->eps > 0.0f)) return fail(MFCC_E_INVALID, "eps must be positive");
    return MFCC_OK;
}

}  // namespace

extern "C" {

int mfcc_causal_conv(const mfcc_conv_args* a, void* stream) try {
    if (const int rc = check_conv(a)) return rc;
    if (a->rows > 0 && (!a->d_x || !a->d_y)) return fail(MFCC_E_INVALID, "NULL convolution buffer");
    return by_type(a->dtype, [&](auto t) { return conv_forward<decltype(t)>(a, static_cast<hipStream_t>(stream)); });
} PACKED_CATCH_ALL

size_t mfcc_causal_conv_backward_workspace(const mfcc_conv_args* a) {
    if (check_conv(a)) return 0;
    return (size_t)conv_bwd_parts(a) * (size_t)(a->width + 1) * (size_t)a->channels * sizeof(float);
}

int mfcc_causal_conv_backward(const mfcc_conv_args* a, void* stream) try {
    if (const int rc = check_conv(a)) return rc;
    if (a->rows > 0 && (!a->d_x || !a->d_dy || !a->d_dx)) return fail(MFCC_E_INVALID, "NULL convolution buffer");
    if (!a->d_dweight) return fail(MFCC_E_INVALID, "NULL dweight");
    const size_t need = mfcc_causal_conv_backward_workspace(a);
    if (need && (a->workspace_bytes < need || !a->d_workspace))
        return fail(MFCC_E_WORKSPACE, "workspace too small (mfcc_causal_conv_backward_workspace)");
    return by_type(a->dtype, [&](auto t) { return conv_backward<decltype(t)>(a, static_cast<hipStream_t>(stream)); });
} PACKED_CATCH_ALL

int mfcc_causal_conv_step(int32_t dtype, int32_t batch, int32_t n_slots, int32_t channels, int32_t width,
                          int32_t activation, const void* d_x, int64_t x_stride, const void* d_state, void* d_new_state,
                          const float* d_weight, const float* d_bias, const int32_t* d_slots, void* d_y, int64_t y_stride,
                          void* stream) try {
    if (batch < 0 || n_slots < 0 || channels < 1 || channels > MAX_CHANNELS) return fail(MFCC_E_INVALID, "bad convolution shape");
    if (width < 1 || width > 8) return fail(MFCC_E_INVALID, "width must lie between 1 and 8");
    if (activation != MFCC_ACT_NONE && activation != MFCC_ACT_SILU) return fail(MFCC_E_INVALID, "unknown activation");
    if (!d_slots && batch > n_slots) return fail(MFCC_E_INVALID, "more entries than states");
    if (batch > 65535) return fail(MFCC_E_UNSUPPORTED, "more than 65535 entries: split the call");
    if (batch == 0) return MFCC_OK;
    if (!d_x || !d_weight || !d_y || (width > 1 && n_slots > 0 && (!d_state || !d_new_state)))
        return fail(MFCC_E_INVALID, "NULL convolution buffer");
    ConvStep f;
    f.x = d_x; f.x_stride = x_stride; f.state = d_state; f.new_state = d_new_state; f.w = d_weight; f.bias = d_bias;
    f.slots = d_slots; f.y = d_y; f.y_stride = y_stride; f.batch = batch; f.n_slots = n_slots; f.channels = channels;
    f.n_vec = 0; f.act = activation == MFCC_ACT_SILU;
    return by_type(dtype, [&](auto t) { return conv_step<decltype(t)>(f, width, static_cast<hipStream_t>(stream)); });
} PACKED_CATCH_ALL

size_t mfcc_selective_scan_workspace(const mfcc_scan_args* a) {
    if (check_scan(a, false)) return 0;
    return scan_space(a, false).total;
}

int mfcc_selective_scan(const mfcc_scan_args* a, void* stream) try {
    if (const int rc = check_scan(a, false)) return rc;
    if (a->rows > 0 && !a->d_y) return fail(MFCC_E_INVALID, "NULL scan buffer");
    const size_t need = scan_space(a, false).total;
    if (need && (a->workspace_bytes < need || !a->d_workspace))
        return fail(MFCC_E_WORKSPACE, "workspace too small (mfcc_selective_scan_workspace)");
    return by_type(a->dtype, [&](auto t) { return scan_forward<decltype(t)>(a, static_cast<hipStream_t>(stream)); });
} PACKED_CATCH_ALL

size_t mfcc_selective_scan_backward_workspace(const mfcc_scan_args* a) {
    if (check_scan(a, false)) return 0;
    return scan_space(a, true).total;
}

int mfcc_selective_scan_backward(const mfcc_scan_args* a, void* stream) try {
    if (const int rc = check_scan(a, false)) return rc;
    if (a->rows > 0 && (!a->d_dy || !a->d_du || !a->d_ddelta || !a->d_dB || !a->d_dC))
        return fail(MFCC_E_INVALID, "NULL scan buffer");
    if (!a->d_dA) return fail(MFCC_E_INVALID, "NULL dA");
    const size_t need = scan_space(a, true).total;
    if (need && (a->workspace_bytes < need || !a->d_workspace))
        return fail(MFCC_E_WORKSPACE, "workspace too small (mfcc_selective_scan_backward_workspace)");
    return by_type(a->dtype, [&](auto t) { return scan_backward<decltype(t)>(a, static_cast<hipStream_t>(stream)); });
} PACKED_CATCH_ALL

int mfcc_selective_scan_step(const mfcc_scan_args* a, int32_t n_slots, const int32_t* d_slots, void* stream) try {
    if (const int rc = check_scan(a, true)) return rc;
    if (n_slots < 0 || (!d_slots && a->rows > n_slots)) return fail(MFCC_E_INVALID, "more entries than states");
    if (a->rows > 65535) return fail(MFCC_E_UNSUPPORTED, "more than 65535 entries: split the call");
    if (a->rows == 0) return MFCC_OK;
    if (!a->d_y || (n_slots > 0 && (!a->d_initial || !a->d_final))) return fail(MFCC_E_INVALID, "NULL scan buffer");
    return by_type(a->dtype, [&](auto t) { return scan_step<decltype(t)>(a, n_slots, d_slots, static_cast<hipStream_t>(stream)); });
} PACKED_CATCH_ALL

int mfcc_add_norm(const mfcc_norm_args* a, void* stream) try {
    if (const int rc = check_norm(a, false)) return rc;
    if (a->rows > 0 && (!a->d_x || !a->d_y)) return fail(MFCC_E_INVALID, "NULL norm buffer");
    return by_type(a->dtype, [&](auto t) { return add_norm_forward<decltype(t)>(a, static_cast<hipStream_t>(stream)); });
} PACKED_CATCH_ALL

int mfcc_gate_norm(const mfcc_norm_args* a, void* stream) try {
    if (const int rc = check_norm(a, true)) return rc;
    if (a->rows > 0 && (!a->d_x || !a->d_z || !a->d_y)) return fail(MFCC_E_INVALID, "NULL norm buffer");
    return by_type(a->dtype, [&](auto t) { return gate_norm_forward<decltype(t)>(a, static_cast<hipStream_t>(stream)); });
} PACKED_CATCH_ALL

size_t mfcc_norm_backward_workspace(const mfcc_norm_args* a) {
    if (check_norm(a, true) && check_norm(a, false)) return 0;
    return norm_bwd_space(a);
}

int mfcc_add_norm_backward(const mfcc_norm_args* a, void* stream) try {
    if (const int rc = check_norm(a, false)) return rc;
    if (a->rows > 0 && (!a->d_r || (a->d_dscale && !a->d_x))) return fail(MFCC_E_INVALID, "NULL norm buffer");
    if ((a->d_dweight || a->d_dbias || a->d_dscale) && a->rows > 0 &&
        (a->workspace_bytes < mfcc_norm_backward_workspace(a) || !a->d_workspace))
        return fail(MFCC_E_WORKSPACE, "workspace too small (mfcc_norm_backward_workspace)");
    return by_type(a->dtype, [&](auto t) { return add_norm_backward<decltype(t)>(a, static_cast<hipStream_t>(stream)); });
} PACKED_CATCH_ALL

int mfcc_gate_norm_backward(const mfcc_norm_args* a, void* stream) try {
    if (const int rc = check_norm(a, true)) return rc;
    if (a->rows > 0 && (!a->d_x || !a->d_z || !a->d_dy || !a->d_dx || !a->d_dz)) return fail(MFCC_E_INVALID, "NULL norm buffer");
    if ((a->d_dweight || a->d_dbias) && a->rows > 0 &&
        (a->workspace_bytes < mfcc_norm_backward_workspace(a) || !a->d_workspace))
        return fail(MFCC_E_WORKSPACE, "workspace too small (mfcc_norm_backward_workspace)");
    return by_type(a->dtype, [&](auto t) { return gate_norm_backward<decltype(t)>(a, static_cast<hipStream_t>(stream)); });
} PACKED_CATCH_ALL

}  // extern "C"
