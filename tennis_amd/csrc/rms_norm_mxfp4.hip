#include "rms_norm.hpp"

namespace tsx {
int rms_norm_mxfp4(const RmsNormParams &p, int type, hipStream_t stream) { return rms_norm_of<NORM_MXFP4>(p, type, stream); }
}
