// One operator family over one element type per translation unit (PACKED_OP, PACKED_TYPE from the Makefile),
// so that they compile side by side.
#if PACKED_TYPE == 0
#define PT F32
#elif PACKED_TYPE == 1
#define PT BF16
#else
#define PT F16
#endif

#if PACKED_OP == 0
#include "packed_conv.h"
namespace packed {
template int conv_forward<PT>(const mfcc_conv_args*, hipStream_t);
template int conv_backward<PT>(const mfcc_conv_args*, hipStream_t);
template int conv_step<PT>(ConvStep, int, hipStream_t);
}
#elif PACKED_OP == 1
#include "packed_scan.h"
namespace packed {
template int scan_forward<PT>(const mfcc_scan_args*, hipStream_t);
template int scan_backward<PT>(const mfcc_scan_args*, hipStream_t);
template int scan_step<PT>(const mfcc_scan_args*, int, const int32_t*, hipStream_t);
}
#else
#include "packed_norm.h"
namespace packed {
template int add_norm_forward<PT>(const mfcc_norm_args*, hipStream_t);
template int add_norm_backward<PT>(const mfcc_norm_args*, hipStream_t);
template int gate_norm_forward<PT>(const mfcc_norm_args*, hipStream_t);
template int gate_norm_backward<PT>(const mfcc_norm_args*, hipStream_t);
}
#endif
