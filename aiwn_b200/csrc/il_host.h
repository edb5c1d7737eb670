// il_host.h -- host helpers shared by the translation units of the library.
#pragma once

namespace il {

// the current device: IL_OK where it is sm_100 (its SM count in *num_sms, unless null), else IL_ERR_DEVICE
__attribute__((visibility("hidden"))) int host_check_device(int* num_sms);

// after a launch of `kernels` kernels: counts them, IL_OK or IL_ERR_LAUNCH
__attribute__((visibility("hidden"))) int host_launch_status(int kernels);

}  // namespace il
