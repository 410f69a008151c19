// Attention of few rows over the 8-bit cache: f16 queries.
#include "tq_attend_few_impl.h"

template int tq::launch_attend_few<TQ_F16, true>(const tq::Attend&, int, unsigned, hipStream_t);
