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
extern template int launch_rows<bf16, float, true>(GroupedArgs, hipStream_t);
extern template int launch_rows<f16, float, true>(GroupedArgs, hipStream_t);

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

namespace face {
// Workspace of the backward: a row of dx per slot where the rows of x are shared, then the weights' partial results. The
// slots' rows are fp32 whatever the rows' type: their sum is rounded once, and a part past fp16's largest is no infinity.
static int64_t slot_rows_bytes(int64_t slots, int32_t k, int32_t x_div) {
    return x_div > 1 ? (slots * k * 4 + 255) / 256 * 256 : 0;
}
static int64_t part_bytes(int64_t slots, int32_t n, int32_t k, int32_t dtype, bool with_bias) {
    // the most shares of the ways the call may go; one group has them wherever several have
    int shares = weight_shares(slots, 1, n, k, dtype, false, false);
    if (dtype != FACE_F32) {
        auto more = [&](bool large) {
            const int s = weight_shares(slots, 1, n, k, dtype, large, true);
            if (s > shares) shares = s;
        };
        more(false);
        if (weight_large(slots, n, k)) more(true);
    }
    return shares > 1 ? 2 * shares * ((int64_t)n * k + (with_bias ? n : 0)) * 4 : 0;
}
}  // namespace face

extern "C" int64_t face_grouped_linear_bwd_work(int64_t slots, int32_t n, int32_t k, int32_t dtype, int32_t x_div,
                                                int32_t with_dx, int32_t with_dw, int32_t with_db) {
    if (slots <= 0 || n <= 0 || k <= 0) return 0;
    return (with_dx ? slot_rows_bytes(slots, k, x_div) : 0) + (with_dw ? part_bytes(slots, n, k, dtype, with_db) : 0);
}

extern "C" int face_grouped_linear_bwd(const void* x, int64_t ld_x, int32_t x_div, int32_t x_op, const void* dy,
                                       int64_t ld_dy, const void* w, int64_t ld_w, int64_t w_group, const int32_t* ptr,
                                       const int32_t* order, int64_t slots, int32_t G, int32_t n, int32_t k, int32_t dtype,
                                       void* dx, void* dw, void* db, void* work, int64_t work_bytes, void* stream) {
    if (int rc = grouped_args(ptr, order, slots, G, n, k, dtype)) return rc;
    if (x_div <= 0 || slots % x_div || (x_op != 0 && x_op != 1) || ld_x < k || ld_dy < n || (db && !dw)) return FACE_ERR_ARG;
    if (dx && (ld_w < k || w_group < 0)) return FACE_ERR_ARG;
    if (dw && !ptr) return FACE_ERR_ARG;
    if (slots && (!dy || (dx && !w) || ((dw || x_op) && !x))) return FACE_ERR_ARG;
    const int64_t need = face_grouped_linear_bwd_work(slots, n, k, dtype, x_div, dx != nullptr, dw != nullptr, db != nullptr);
    if (work_bytes < need || (need && !work)) return FACE_ERR_ARG;
    char* part = (char*)work + (dx ? slot_rows_bytes(slots, k, x_div) : 0);
    const hipStream_t st = (hipStream_t)stream;
    if (dx && slots) {
        void* rows = x_div > 1 ? work : dx;
        GroupedArgs g = {dy, ld_dy, 1, 0, w, ld_w, w_group, nullptr, 0, nullptr, nullptr, rows, k, x_op ? x : nullptr, ld_x,
                         x_div, k, n, ptr, order, slots, G, 0, 0};
        int rc = with_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            return x_div > 1 ? launch_rows<T, float, true>(g, st) : launch_rows<T, T, true>(g, st);
        });
        if (!rc && x_div > 1) rc = sum_slot_rows((const float*)work, slots / x_div, x_div, k, dtype, dx, st);
        if (rc) return rc;
    }
    if (dw) {
        GroupedWArgs g = {x, ld_x, x_div, x_op, 0, 0, dy, ld_dy, dw, db, (float*)part, n, k, ptr, order, slots, G, 0, 0, 0, 0};
        return with_dtype(dtype, [&](auto t) { return launch_weight<decltype(t)>(g, st); });
    }
    return 0;
}
