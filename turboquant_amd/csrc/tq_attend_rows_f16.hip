// Attention of many rows over exact blocks: f16 queries.
#include "tq_attend_rows_impl.h"

template int tq::launch_attend_rows<TQ_F16, false>(const tq::Attend&, unsigned, hipStream_t);
