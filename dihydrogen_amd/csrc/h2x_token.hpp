// What the token operators (layer normalisation, rotary positions, attention) share: element types, rows of strided
// tensors, sums over a wave in the type they are held in.
#pragma once

#include "h2x_device.hpp"

namespace h2x
{
namespace token
{

using bf16 = __bf16;
using f16 = _Float16;

inline int element_size(int dtype)
{
    switch (dtype)
    {
    case H2X_F32: return 4;
    case H2X_F64: return 8;
    case H2X_BF16:
    case H2X_F16: return 2;
    default: return 0;
    }
}

// Sums of rows are held in 32 bits, those of doubles in 64.
template <typename T>
struct Wide
{
    using type = float;
};
template <>
struct Wide<double>
{
    using type = double;
};
template <typename T>
using wide = typename Wide<T>::type;

// Rows of a tensor, at most five dimensions besides the innermost one: row r lies at offset(r) elements.
constexpr int kMaxOuter = H2X_MAX_DIMS - 1;
struct Rows
{
    int64_t stride[kMaxOuter]; // of the dimensions, the first of which runs fastest
    FastDiv extent[kMaxOuter];
    int num; // 0: rows one after another, stride[0] apart
};

// Whether two tensors' rows lie alike.
inline bool alike(const Rows& a, const Rows& b)
{
    if (a.num != b.num || a.stride[0] != b.stride[0])
        return false;
    for (int d = 0; d < a.num; ++d)
        if (a.stride[d] != b.stride[d] || a.extent[d].divisor != b.extent[d].divisor)
            return false;
    return true;
}

#ifdef __HIPCC__
__device__ __forceinline__ int64_t row_offset(const Rows& rows, uint32_t r)
{
    if (rows.num == 0)
        return static_cast<int64_t>(r) * rows.stride[0];
    int64_t at = 0;
    for (int d = 0; d + 1 < rows.num; ++d)
    {
        const uint32_t q = fastdiv(r, rows.extent[d]);
        at += static_cast<int64_t>(r - q * rows.extent[d].divisor) * rows.stride[d];
        r = q;
    }
    return at + static_cast<int64_t>(r) * rows.stride[rows.num - 1];
}

__device__ __forceinline__ float wave_total(float v)
{
    return wave_combine(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ double wave_total(double v)
{
    return wave_combine(v, [](double a, double b) { return a + b; });
}
#endif

// False: not rows of `channels` elements, as many as said.
inline bool make_rows(const h2x_tensor_geometry* g, size_t num_rows, int channels, Rows* out)
{
    *out = Rows{};
    out->stride[0] = channels;
    if (!g)
        return true;
    if (g->num_dims < 1 || g->num_dims > H2X_MAX_DIMS || g->local_shape[0] != channels || g->strides[0] != 1)
        return false;
    uint64_t rows = 1;
    for (int d = 1; d < g->num_dims; ++d)
    {
        if (g->local_shape[d] < 0 || g->local_shape[d] > 0x7fffffff)
            return false;
        rows *= static_cast<uint64_t>(g->local_shape[d]);
        if (rows > 0x7fffffffu)
            return false;
    }
    if (rows != num_rows)
        return false;
    if (rows == 0)
        return true;
    // dimensions that go on where the one inside them ends are one
    int n = 0;
    int64_t extents[kMaxOuter];
    for (int d = 1; d < g->num_dims; ++d)
    {
        if (g->local_shape[d] == 1)
            continue;
        if (n > 0 && g->strides[d] == out->stride[n - 1] * extents[n - 1])
        {
            extents[n - 1] *= g->local_shape[d];
            continue;
        }
        extents[n] = g->local_shape[d];
        out->stride[n++] = g->strides[d];
    }
    if (n == 0) // one row
        out->stride[0] = channels;
    for (int d = 0; d < n; ++d)
        out->extent[d] = make_fastdiv(static_cast<uint32_t>(extents[d]));
    out->num = n > 1 ? n : 0;
    return true;
}

} // namespace token
} // namespace h2x
