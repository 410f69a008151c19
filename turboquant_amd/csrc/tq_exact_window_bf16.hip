// A window's weights over a paged exact cache: the kernels for bf16 elements.
#include "tq_exact_window_impl.h"

template int tq::launch_exact_window<TQ_BF16>(const tq::ExactWindow&, bool, hipStream_t);
