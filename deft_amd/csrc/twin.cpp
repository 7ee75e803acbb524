// The `_p3` entry points of sources whose code does not depend on the operand pieces (rotary.hip, attn.hip): the same kernels, the refusal's text in the `_p3`
// set's error string.  Linked where both sets are in one library (deft_amd/build.py).
#include "../../include/deft_hip.h"

void deft_set_error_p3(const char* fmt, ...) __asm__("_Z14deft_set_errorPKcz_p3");      // csrc/ops.hip's, as the build renames it

namespace {
template <typename R>
R told(R rc) {
    if (rc < 0) deft_set_error_p3("%s", deft_last_error());
    return rc;
}
}  // namespace

extern "C" int deft_rotary_p3(const DeftRotary* d, void* stream) { return told(deft_rotary(d, stream)); }
extern "C" int deft_attn_p3(const DeftAttn* d, void* stream) { return told(deft_attn(d, stream)); }
extern "C" long long deft_attn_ws_floats_p3(const DeftAttn* d) { return told(deft_attn_ws_floats(d)); }
