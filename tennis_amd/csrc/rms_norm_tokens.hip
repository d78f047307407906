#include "rms_norm.hpp"

namespace tsx {
int rms_norm_tokens(const RmsNormParams &p, int type, hipStream_t stream) { return rms_norm_of<NORM_TOKENS>(p, type, stream); }
}
