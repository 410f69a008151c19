// A window's weights over a paged exact cache: the kernels for fp32 elements.
#include "tq_exact_window_impl.h"

template int tq::launch_exact_window<TQ_F32>(const tq::ExactWindow&, bool, hipStream_t);
