// libophelia_seq.so -- errors and devices of its C entry points.
#include <stdarg.h>
#include <stdio.h>

#include "oph_seq.h"
#include "../../include/ophelia_hip.h"

namespace ophseq {

static thread_local char g_error[256] = "";

int fail(int status, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof g_error, fmt, ap);
    va_end(ap);
    return status;
}

int type_bytes(int dtype) { return dtype == OPH_SEQ_F32 ? 4 : dtype == OPH_SEQ_BF16 || dtype == OPH_SEQ_F16 ? 2 : 0; }

// An error of the runtime goes to the caller as this call's, and is taken from the runtime: its next reader would report it as its own.
int device_fail(hipError_t e, const char* what) {
    (void)hipGetLastError();
    return fail(OPH_ERR_DEVICE, "%s: %s", what, hipGetErrorString(e));
}

OnDevice::OnDevice(int device) {
    int now = -1;
    if (hipError_t e = hipGetDevice(&now)) { status = device_fail(e, "no usable HIP device (no CPU fallback)"); return; }
    if (now == device) return;
    if (device < 0) { status = fail(OPH_ERR_DEVICE, "device %d cannot be used", device); return; }
    if (hipError_t e = hipSetDevice(device)) { status = device_fail(e, "the device cannot be used"); return; }
    before = now;
}
OnDevice::~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
}

}  // namespace ophseq

extern "C" {
int oph_seq_abi_version(void) { return OPH_SEQ_ABI_VERSION; }
const char* oph_seq_last_error(void) { return ophseq::g_error; }
}
