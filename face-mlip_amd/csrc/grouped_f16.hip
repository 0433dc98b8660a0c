// The grouped products of f16 rows.
#include "grouped.h"

namespace face {
template int launch_rows<f16, f16, false>(GroupedArgs, hipStream_t);
template int launch_rows<f16, f16, true>(GroupedArgs, hipStream_t);
template int launch_rows<f16, float, true>(GroupedArgs, hipStream_t);
template int launch_weight<f16>(GroupedWArgs, hipStream_t);
}  // namespace face
