// Attention of few rows over exact blocks: bf16 queries.
#include "tq_attend_few_impl.h"

template int tq::launch_attend_few<TQ_BF16, false>(const tq::Attend&, int, unsigned, hipStream_t);
