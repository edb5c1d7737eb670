// il_host.h -- host helpers shared by the translation units of the library.
#pragma once
#include <stddef.h>

namespace il {

// the current device: IL_OK where it is sm_100 (its SM count in *num_sms, unless null), else IL_ERR_DEVICE
__attribute__((visibility("hidden"))) int host_check_device(int* num_sms);

// after a launch of `kernels` kernels: counts them, IL_OK or IL_ERR_LAUNCH
__attribute__((visibility("hidden"))) int host_launch_status(int kernels);

// Before a launch of `kern` with smem bytes of dynamic shared memory.  What a kernel may have belongs to the kernel and
// the device, not to a launch: set to a call's own size, another host thread's smaller one between the two would make
// the launch fail.  So it is set once, to all that the kernel's static arrays leave, and never lowered.
__attribute__((visibility("hidden"))) int host_allow_shared(const void* kern, size_t smem);

}  // namespace il
