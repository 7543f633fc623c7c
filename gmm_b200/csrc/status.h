// status.h -- what the library's source files share on the host: the calling
// thread's error text (gmm_sm100_last_error) and the current device's size.
#pragma once

namespace gmm_sm100 {

// Records `msg` as this thread's last error and returns `code`.
int set_error(int code, const char* msg) noexcept;

// SM count of the current device; a status if it is not a B200-class GPU.
int current_sm_count(int* sms);

// The norm and quantiser kernels' parts of gmm_sm100_device_error.
int norm_fwd_device_error(int* status, bool clear);
int norm_bwd_device_error(int* status, bool clear);
int quant_device_error(int* status, bool clear);

}  // namespace gmm_sm100
