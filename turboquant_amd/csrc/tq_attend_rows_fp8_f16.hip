// Attention of many rows over the 8-bit cache: f16 queries.
#include "tq_attend_rows_impl.h"

template int tq::launch_attend_rows<TQ_F16, true>(const tq::Attend&, unsigned, hipStream_t);
