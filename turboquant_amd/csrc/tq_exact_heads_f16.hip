// Decode attention over a paged exact cache, dozens of query heads on a KV head: the kernels for fp16 elements.
#include "tq_exact_heads_impl.h"

template int tq::launch_exact_heads<TQ_F16>(const tq::ExactDecode&, hipStream_t);
