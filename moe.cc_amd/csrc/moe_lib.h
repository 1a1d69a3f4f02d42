// moe_lib.h - library-internal helpers shared by the C ABI translation units.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/moehip.h"

namespace moe {
// Records a message for moe_last_error() and returns `st`.
moe_status set_error(moe_status st, const char* fmt, ...);
// MOE_OK, or MOE_ERR_HIP with "<what>: <hip error string>" recorded.
moe_status check_hip(hipError_t e, const char* what);
// Initialises device 0 if moe_init has not been called.
moe_status ensure_init();
// The library's stream.
hipStream_t stream();
// The device it belongs to (-1 before initialisation).
int device();
// Work is queued on the library's stream whatever device the calling thread
// has current.
struct OnDevice {
  int was = -1;
  moe_status enter() {
    int d = -1;
    moe_status st = check_hip(hipGetDevice(&d), "hipGetDevice");
    if (st || d == device()) return st;
    was = d;
    return check_hip(hipSetDevice(device()), "hipSetDevice");
  }
  ~OnDevice() {
    if (was >= 0) (void)hipSetDevice(was);
  }
};
// Layers and models alive (moe_shutdown refuses while any is).
void live_objects(int delta);
// The scratch of a layer's forward over T rows, so that the forward allocates none.
moe_status reserve_layer(moe_layer* layer, int T);
// Free the library-owned device buffers of one translation unit (the
// stream has drained; called by moe_shutdown only).
void release_gemv_workspace();
void release_layer_scratch();
}  // namespace moe
