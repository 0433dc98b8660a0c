// The grouped products of e4m3 rows (forward only), results in fp32, bf16 or fp16.
#include "grouped.h"

namespace face {
template int launch_rows<e4m3_wide, float, false>(GroupedArgs, hipStream_t);
template int launch_rows<e4m3, bf16, false>(GroupedArgs, hipStream_t);
template int launch_rows<e4m3, f16, false>(GroupedArgs, hipStream_t);
}  // namespace face
