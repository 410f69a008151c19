// Decode attention over a paged exact cache: the page-streaming kernel for bf16 elements.
#include "tq_exact_impl.h"

template int tq::launch_exact_decode<TQ_BF16>(const tq::ExactDecode&, hipStream_t);
