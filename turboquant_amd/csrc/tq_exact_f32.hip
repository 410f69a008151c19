// Decode attention over a paged exact cache: the page-streaming kernel for fp32 elements.
#include "tq_exact_impl.h"

template int tq::launch_exact_decode<TQ_F32>(const tq::ExactDecode&, hipStream_t);
