// Rotary positions with several axes (include/h2x.h has the definition).
//
// Bound by memory: every element is read and written once.  An angle belongs to a token and a pair, not to a head, so a
// thread makes the sine and cosine of its pairs once and turns the same pairs of many heads with them.  Angles are made in 64
// bits and brought to a fraction of a turn there: at position 2^20 an angle in 32 bits is off by 0.06.  Sine and cosine of that
// are taken in 32 bits (64 for doubles).
#include "h2x_token.hpp"

namespace h2x
{
namespace token
{
namespace
{

struct Turn
{
    const int32_t* positions;
    const double* frequencies;
    int64_t positions_sample_stride, positions_axis_stride;
    int32_t axis_end[H2X_MAX_AXES]; // pairs up to the end of each axis
    int32_t pairs, head_dim, heads, neighbours;
    double sign;
    int64_t tokens;
    h2x_token_strides x, y;
    // a workgroup: `columns` threads side by side, each with V pairs of a token (or V elements that are copied), by `rows`, each with
    // a token of its own
    FastDiv columns;
    int32_t rows, vectors; // vectors of V pairs in the turned part
    int32_t head_groups;   // workgroups that share a token's heads
    uint32_t token_groups; // workgroups side by side along the tokens
    FastDiv by_head_groups;
    uint64_t first; // workgroups before the launch
};

// Sine and cosine of position * frequency.  At positions of 31 bits a rounding of the angle, or of the turns that it makes, is 2^-25 of a turn and
// more, three steps of a sine: the product and 1 / (2 pi) are taken in two numbers each.  What is left, within half a turn, fits 32 bits to
// 2^-26 of a turn (a sine of 1.6 * 2^-24); the part that does not, x, is turned by after sine and cosine: s + x c and c - x s, whose next terms are x^2 /
// 2 = 2^-48.
__device__ __forceinline__ void sine_cosine(double position, double frequency, float* s, float* c)
{
    constexpr double kPerTurn = 0.15915494309189535, kPerTurnRest = -9.839338337591243e-18; // 1 / (2 pi)
    const double angle = position * frequency, angle_rest = __builtin_fma(position, frequency, -angle);
    const double whole = rint(angle * kPerTurn);
    const double turns = __builtin_fma(angle, kPerTurn, -whole) + __builtin_fma(angle, kPerTurnRest, angle_rest * kPerTurn);
    const float rest = static_cast<float>(turns), x = static_cast<float>((turns - rest) * 6.283185307179586);
    float sine, cosine;
    sincospif(2.0f * rest, &sine, &cosine);
    *s = __builtin_fmaf(x, cosine, sine);
    *c = __builtin_fmaf(-x, sine, cosine);
}
__device__ __forceinline__ void sine_cosine(double position, double frequency, double* s, double* c)
{
    sincos(position * frequency, s, c);
}

template <typename W>
__device__ __forceinline__ W fused(W a, W b, W c)
{
    if constexpr (sizeof(W) == 8)
        return __builtin_fma(a, b, c);
    else
        return __builtin_fmaf(a, b, c);
}

// V pairs a thread: V = elements of 16 bytes, of which the pairs are halves (two loads) or neighbours (two loads side by
// side), of 8 bytes, or 1 where strides, sizes or addresses are no multiples of that.  Two samples of 16 x 32 x 32 tokens, 32 heads of 128 in
// bf16, three axes: 116 us, 4.6 TB/s of the 5.1 that a copy reaches.
template <typename T, int V, bool Neighbours>
__global__ void __launch_bounds__(kBlockSize) rotary_kernel(const T* x, T* y, const Turn a)
{
    using W = wide<T>;
    using Vec = AVec<T, V>;
    const uint32_t row = fastdiv(threadIdx.x, a.columns), column = threadIdx.x - row * a.columns.divisor;
    if (row >= static_cast<uint32_t>(a.rows))
        return;
    const uint64_t group = a.first + blockIdx.x;
    const uint64_t token_group = group / a.head_groups;
    const int head_group = static_cast<int>(group - token_group * a.head_groups);
    const int64_t sample = token_group / a.token_groups;
    const int64_t token = static_cast<int64_t>(token_group - sample * a.token_groups) * a.rows + row;
    if (token >= a.tokens)
        return;
    x += sample * a.x.sample + token * a.x.token;
    y += sample * a.y.sample + token * a.y.token;
    const int vector = column;
    if (vector < a.vectors)
    {
        W s[V], c[V];
        const int pair = vector * V;
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
            int axis = 0;
#pragma unroll
            for (int n = 0; n < H2X_MAX_AXES - 1; ++n)
                axis += pair + i >= a.axis_end[n];
            const double position =
                a.positions[sample * a.positions_sample_stride + axis * a.positions_axis_stride + token];
            sine_cosine(a.sign * position, a.frequencies[pair + i], &s[i], &c[i]);
        }
        const int first = Neighbours ? 2 * pair : pair, second = Neighbours ? 2 * pair + V : pair + a.pairs;
        for (int h = head_group; h < a.heads; h += a.head_groups)
        {
            const Vec p = *reinterpret_cast<const Vec*>(x + h * a.x.head + first);
            const Vec q = *reinterpret_cast<const Vec*>(x + h * a.x.head + second);
            Vec to_p, to_q;
            if constexpr (Neighbours && V > 1)
            {
                // p holds pairs 0 .. V / 2 - 1, q the others
#pragma unroll
                for (int i = 0; i < V; ++i)
                {
                    const Vec& from = i < V / 2 ? p : q;
                    Vec& to = i < V / 2 ? to_p : to_q;
                    const int at = 2 * (i % (V / 2));
                    const W u = static_cast<W>(from.v[at]), v = static_cast<W>(from.v[at + 1]);
                    to.v[at] = static_cast<T>(fused(u, c[i], -(v * s[i])));
                    to.v[at + 1] = static_cast<T>(fused(u, s[i], v * c[i]));
                }
            }
            else
            {
#pragma unroll
                for (int i = 0; i < V; ++i)
                {
                    const W u = static_cast<W>(p.v[i]), v = static_cast<W>(q.v[i]);
                    to_p.v[i] = static_cast<T>(fused(u, c[i], -(v * s[i])));
                    to_q.v[i] = static_cast<T>(fused(u, s[i], v * c[i]));
                }
            }
            *reinterpret_cast<Vec*>(y + h * a.y.head + first) = to_p;
            *reinterpret_cast<Vec*>(y + h * a.y.head + second) = to_q;
        }
    }
    else
    {
        const int at = 2 * a.pairs + (vector - a.vectors) * V;
        for (int h = head_group; h < a.heads; h += a.head_groups)
            *reinterpret_cast<Vec*>(y + h * a.y.head + at) = *reinterpret_cast<const Vec*>(x + h * a.x.head + at);
    }
}

// Whether every vector of V elements lies on a multiple of its size.
template <int V>
bool whole_vectors(const void* p, const h2x_token_strides& s, size_t size)
{
    return reinterpret_cast<uintptr_t>(p) % (V * size) == 0 && s.sample % V == 0 && s.token % V == 0 && s.head % V == 0;
}

template <typename T, int V, bool Neighbours>
int issue(const h2x_rotary& r, Turn a, const void* x, void* y, hipStream_t stream)
{
    a.vectors = a.pairs / V;
    const bool copies = x != y; // in place the rest stays where it is
    const int columns = a.vectors + (copies ? (r.head_dim - 2 * a.pairs) / V : 0);
    if (columns == 0)
        return H2X_SUCCESS;
    a.columns = make_fastdiv(columns);
    a.rows = kBlockSize / columns;
    const uint64_t token_groups = (static_cast<uint64_t>(r.tokens) + a.rows - 1) / a.rows;
    a.token_groups = static_cast<uint32_t>(token_groups);
    // A thread turns the heads of its token one after another; fewer each while there are not workgroups for
    // eight a CU, down to two heads a thread.
    a.head_groups = 1;
    while (token_groups * r.samples * a.head_groups < 8 * chip_units() && 2 * a.head_groups <= (r.heads + 1) / 2)
        a.head_groups *= 2;
    const uint64_t groups = token_groups * r.samples * a.head_groups;
    constexpr uint64_t kMost = 0x80000000u / kBlockSize;
    for (a.first = 0; a.first < groups; a.first += kMost)
        launch(rotary_kernel<T, V, Neighbours>, dim3(static_cast<uint32_t>(groups - a.first < kMost ? groups - a.first : kMost)),
               dim3(kBlockSize), stream, static_cast<const T*>(x), static_cast<T*>(y), a);
    return launch_status();
}

template <typename T>
int apply(const h2x_rotary& r, const Turn& a, const void* x, void* y, hipStream_t stream)
{
    // vectors of 16 bytes, of 8 where the sizes allow no more (heads of 72 with all 36 pairs in bf16), or single elements
    const auto fits = [&](auto v) {
        constexpr int V = decltype(v)::value;
        return whole_vectors<V>(x, r.x, sizeof(T)) && whole_vectors<V>(y, r.y, sizeof(T)) && a.pairs % V == 0 && r.head_dim % V == 0;
    };
    const auto by_pairing = [&](auto v) {
        constexpr int V = decltype(v)::value;
        return a.neighbours ? issue<T, V, true>(r, a, x, y, stream) : issue<T, V, false>(r, a, x, y, stream);
    };
    constexpr std::integral_constant<int, 16 / sizeof(T)> whole;
    constexpr std::integral_constant<int, 8 / sizeof(T)> half;
    if (fits(whole))
        return by_pairing(whole);
    if (sizeof(T) < 8 && fits(half))
        return by_pairing(half);
    return by_pairing(std::integral_constant<int, 1>());
}

} // namespace
} // namespace token
} // namespace h2x

using namespace h2x;
using namespace h2x::token;

extern "C" int h2x_rotary_apply(const h2x_rotary* rotary, const void* x, const int32_t* positions, const double* frequencies,
                                int inverse, void* y, h2x_stream_t stream)
{
    if (!rotary)
        return H2X_ERR_INVALID_ARGUMENT;
    const h2x_rotary& r = *rotary;
    if (element_size(r.dtype) == 0)
        return H2X_ERR_UNSUPPORTED;
    if (r.head_dim < 1 || r.heads < 0 || r.samples < 0 || r.tokens < 0 || r.num_axes < 0 || r.num_axes > H2X_MAX_AXES
        || (r.pairing != H2X_ROTARY_HALVES && r.pairing != H2X_ROTARY_NEIGHBOURS))
        return H2X_ERR_INVALID_ARGUMENT;
    Turn a{};
    int64_t pairs = 0;
    for (int n = 0; n < H2X_MAX_AXES; ++n)
    {
        if (n < r.num_axes)
        {
            if (r.axis_pairs[n] < 0)
                return H2X_ERR_INVALID_ARGUMENT;
            pairs += r.axis_pairs[n];
        }
        if (2 * pairs > r.head_dim)
            return H2X_ERR_INVALID_ARGUMENT;
        // (axes behind the last one begin where no pair is)
        a.axis_end[n] = n + 1 < r.num_axes ? static_cast<int32_t>(pairs) : r.head_dim;
    }
    if (r.head_dim > kBlockSize)
        return H2X_ERR_UNSUPPORTED;
    if (r.tokens > 0x7fffffff)
        return H2X_ERR_TOO_LARGE;
    if (r.heads == 0 || r.samples == 0 || r.tokens == 0)
        return H2X_SUCCESS;
    if (!x || !y || (pairs > 0 && (!positions || !frequencies)))
        return H2X_ERR_INVALID_ARGUMENT;
    if (x == y && ((r.samples > 1 && r.x.sample != r.y.sample) || (r.tokens > 1 && r.x.token != r.y.token)
                   || (r.heads > 1 && r.x.head != r.y.head)))
        return H2X_ERR_INVALID_ARGUMENT;
    a.positions = positions;
    a.frequencies = frequencies;
    a.positions_sample_stride = r.positions_sample_stride;
    a.positions_axis_stride = r.positions_axis_stride;
    a.pairs = static_cast<int32_t>(pairs);
    a.head_dim = r.head_dim;
    a.heads = r.heads;
    a.neighbours = r.pairing == H2X_ROTARY_NEIGHBOURS;
    a.sign = inverse ? -1.0 : 1.0;
    a.tokens = r.tokens;
    a.x = r.x;
    a.y = r.y;
    switch (r.dtype)
    {
    case H2X_F32: return apply<float>(r, a, x, y, as_stream(stream));
    case H2X_F64: return apply<double>(r, a, x, y, as_stream(stream));
    case H2X_BF16: return apply<bf16>(r, a, x, y, as_stream(stream));
    default: return apply<f16>(r, a, x, y, as_stream(stream));
    }
}
