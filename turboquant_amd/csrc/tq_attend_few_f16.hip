// Attention of few rows over exact blocks: f16 queries.
#include "tq_attend_few_impl.h"

template int tq::launch_attend_few<TQ_F16, false>(const tq::Attend&, int, unsigned, hipStream_t);
