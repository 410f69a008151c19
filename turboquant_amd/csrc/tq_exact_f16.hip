// Decode attention over a paged exact cache: the page-streaming kernel for fp16 elements.
#include "tq_exact_impl.h"

template int tq::launch_exact_decode<TQ_F16>(const tq::ExactDecode&, hipStream_t);
