// The grouped products of f32 rows.
#include "grouped.h"

namespace face {
template int launch_rows<float, float, false>(GroupedArgs, hipStream_t);
template int launch_rows<float, float, true>(GroupedArgs, hipStream_t);
template int launch_weight<float>(GroupedWArgs, hipStream_t);
}  // namespace face
