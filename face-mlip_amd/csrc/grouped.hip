// C entries of the grouped products (grouped.h).
#include <type_traits>

#include "grouped.h"

namespace face {
template <typename Out>
using q8_rows = std::conditional_t<std::is_same_v<Out, float>, e4m3_wide, e4m3>;

#define FACE_GROUPED(T_)                                                                \
    extern template int launch_rows<T_, T_, false>(GroupedArgs, hipStream_t);           \
    extern template int launch_rows<T_, T_, true>(GroupedArgs, hipStream_t);            \
    extern template int launch_weight<T_>(GroupedWArgs, hipStream_t);                   \
    extern template int launch_rows<q8_rows<T_>, T_, false>(GroupedArgs, hipStream_t);
FACE_GROUPED(float)
FACE_GROUPED(bf16)
FACE_GROUPED(f16)
#undef FACE_GROUPED

static int grouped_args(const void* ptr, const void* order, int64_t slots, int32_t G, int32_t n, int32_t k, int32_t dtype) {
    if (slots < 0 || G <= 0 || n <= 0 || k <= 0) return FACE_ERR_ARG;
    if (dtype != FACE_F32 && dtype != FACE_BF16 && dtype != FACE_F16) return FACE_ERR_ARG;
    if (slots >= ((int64_t)1 << 31) || G > 65535 || n > (1 << 30) || k > (1 << 30)) return FACE_ERR_UNSUPPORTED;
    if (slots && (!ptr || !order)) return FACE_ERR_ARG;
    return 0;
}

}  // namespace face

using namespace face;

extern "C" int face_grouped_linear(const void* x, int64_t ld_x, int32_t x_div, int32_t x_op, const void* w, int64_t ld_w,
                                   int64_t w_group, const void* bias, int64_t ld_b, const int32_t* ptr,
                                   const int32_t* order, int64_t slots, int32_t G, int32_t n, int32_t k, int32_t dtype,
                                   void* y, int64_t ld_y, void* stream) {
    if (int rc = grouped_args(ptr, order, slots, G, n, k, dtype)) return rc;
    if (x_div <= 0 || (x_op != 0 && x_op != 1) || ld_x < k || ld_w < k || w_group < 0 || (bias && ld_b < 0) || ld_y < n)
        return FACE_ERR_ARG;
    if (slots == 0) return 0;
    if (!x || !w || !y) return FACE_ERR_ARG;
    GroupedArgs g = {x, ld_x, x_div, x_op, w, ld_w, w_group, bias, ld_b, nullptr, nullptr, y, ld_y, nullptr, 0, 1,
                     n, k, ptr, order, slots, G, 0, 0};
    return with_dtype(dtype, [&](auto t) { return launch_rows<decltype(t), decltype(t), false>(g, (hipStream_t)stream); });
}

extern "C" int face_grouped_linear_q8(const void* x, int64_t ld_x, const float* x_scale, int32_t x_div, const void* w,
                                      int64_t ld_w, int64_t w_group, const float* w_scale, const void* bias, int64_t ld_b,
                                      const int32_t* ptr, const int32_t* order, int64_t slots, int32_t G, int32_t n,
                                      int32_t k, int32_t dtype, void* y, int64_t ld_y, void* stream) {
    if (int rc = grouped_args(ptr, order, slots, G, n, k, dtype)) return rc;
    if (x_div <= 0 || ld_x < k || ld_w < k || w_group < 0 || (bias && ld_b < 0) || ld_y < n) return FACE_ERR_ARG;
    if (slots == 0) return 0;
    if (!x || !w || !y || !x_scale || !w_scale) return FACE_ERR_ARG;
    GroupedArgs g = {x, ld_x, x_div, 0, w, ld_w, w_group, bias, ld_b, x_scale, w_scale, y, ld_y, nullptr, 0, 1,
                     n, k, ptr, order, slots, G, 0, 0};
    return with_dtype(dtype, [&](auto t) { return launch_rows<q8_rows<decltype(t)>, decltype(t), false>(g, (hipStream_t)stream); });
}

extern "C" int face_grouped_linear_dx(const void* dy, int64_t ld_dy, const void* w, int64_t ld_w, int64_t w_group,
                                      const void* z, int64_t ld_z, int32_t z_div, const int32_t* ptr, const int32_t* order,
                                      int64_t slots, int32_t G, int32_t n, int32_t k, int32_t dtype, void* dx,
                                      int64_t ld_dx, void* stream) {
    if (int rc = grouped_args(ptr, order, slots, G, n, k, dtype)) return rc;
    if (ld_dy < n || ld_w < k || w_group < 0 || (z && (ld_z < k || z_div <= 0)) || ld_dx < k) return FACE_ERR_ARG;
    if (slots == 0) return 0;
    if (!dy || !w || !dx) return FACE_ERR_ARG;
    GroupedArgs g = {dy, ld_dy, 1, 0, w, ld_w, w_group, nullptr, 0, nullptr, nullptr, dx, ld_dx, z, ld_z, z ? z_div : 1,
                     k, n, ptr, order, slots, G, 0, 0};
    return with_dtype(dtype, [&](auto t) { return launch_rows<decltype(t), decltype(t), true>(g, (hipStream_t)stream); });
}

extern "C" int64_t face_grouped_linear_dw_work(int64_t slots, int32_t n, int32_t k, int32_t dtype, int32_t with_bias) {
    if (slots <= 0 || n <= 0 || k <= 0) return 0;
    const int shares = weight_shares(slots, n, k, dtype);
    return shares > 1 ? 2 * shares * ((int64_t)n * k + (with_bias ? n : 0)) * 4 : 0;
}

extern "C" int face_grouped_linear_dw(const void* x, int64_t ld_x, int32_t x_div, int32_t x_op, const void* dy,
                                      int64_t ld_dy, const int32_t* ptr, const int32_t* order, int64_t slots, int32_t G,
                                      int32_t n, int32_t k, int32_t dtype, void* dw, void* db, void* work,
                                      int64_t work_bytes, void* stream) {
    if (int rc = grouped_args(ptr, order, slots, G, n, k, dtype)) return rc;
    if (x_div <= 0 || (x_op != 0 && x_op != 1) || ld_x < k || ld_dy < n || !ptr || !dw) return FACE_ERR_ARG;
    if (slots && (!x || !dy)) return FACE_ERR_ARG;
    const int64_t need = face_grouped_linear_dw_work(slots, n, k, dtype, db != nullptr);
    if (work_bytes < need || (need && !work)) return FACE_ERR_ARG;
    const int shares = weight_shares(slots, n, k, dtype);
    GroupedWArgs g = {x, ld_x, x_div, x_op, 0, 0, dy, ld_dy, dw, db, (float*)work, n, k, ptr, order, slots, G, 0, 0,
                      shares, (slots + shares - 1) / shares};
    return with_dtype(dtype, [&](auto t) { return launch_weight<decltype(t)>(g, (hipStream_t)stream); });
}
