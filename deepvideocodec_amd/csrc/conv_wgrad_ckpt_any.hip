// The forms of conv_wgrad_ckpt_impl.h for planes whose rows start anywhere (their own translation unit: compile time).
#include "conv_wgrad_ckpt_impl.h"

namespace dvc_wgrad_ckpt {
int launch_any(int ks, int stride, const Args& a, const Plan& p, hipStream_t st) { return launch_shape<false>(ks, stride, a, p, st); }
}  // namespace dvc_wgrad_ckpt
