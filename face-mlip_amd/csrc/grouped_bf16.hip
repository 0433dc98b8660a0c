// The grouped products of bf16 rows.
#include "grouped.h"

namespace face {
template int launch_rows<bf16, bf16, false>(GroupedArgs, hipStream_t);
template int launch_rows<bf16, bf16, true>(GroupedArgs, hipStream_t);
template int launch_rows<bf16, float, true>(GroupedArgs, hipStream_t);
template int launch_weight<bf16>(GroupedWArgs, hipStream_t);
}  // namespace face
