// Layers for grids whose cells are tokens: layer normalisation, rotary positions,
// attention, over the C ABI (include/h2x.h, where the formulas and what is
// refused stand).  The reference has no counterpart.  Layer normalisation takes the framework's
// tensors, the channel innermost (dimension 0), haloed ones by their interior;
// rotary positions and attention take device pointers and the structures of
// the C ABI, whose element types include the 16-bit ones that no tensor here has.
//
// As with the other layers calls are asynchronous on the backend's stream, and an object
// keeps the workspace of its calls: one object is not for two streams, nor for two graphs that run at a time.
#pragma once

#include "distconv/layers_mi355x.hpp"

#include <algorithm>
#include <cmath>
#include <list>
#include <vector>

namespace distconv
{

// A layer's workspace.  One that has become too small is kept until the layer goes: graphs that were captured with it hold its address.  (Each is half as
// large again as the one before at least, so that all of them are three times the last at most.)
class TokenWorkspace
{
public:
    void* get(size_t bytes)
    {
        if (bytes == 0)
            return nullptr;
        const size_t last = m_all.empty() ? 0 : m_all.back().get_size();
        if (last < bytes)
        {
            m_all.emplace_back();
            m_all.back().allocate(std::max(bytes, last + last / 2));
        }
        return m_all.back().get();
    }

private:
    std::list<tensor::Memory<tensor::CUDAAllocator>> m_all;
};

template <typename Backend>
class LayerNormalization;

template <>
class LayerNormalization<BackendMI355X>
{
public:
    explicit LayerNormalization(BackendMI355X const& backend, double epsilon = 1e-5)
        : m_stream(backend.get_stream()), m_epsilon(epsilon)
    {}

    // scale, bias: one element a channel, or nullptr; mean, rstd: one a row, or both nullptr.
    template <typename Tensor>
    int forward(const Tensor& input, const typename Tensor::data_type* scale, const typename Tensor::data_type* bias, Tensor& output,
                typename Tensor::data_type* mean = nullptr, typename Tensor::data_type* rstd = nullptr)
    {
        const h2x_tensor_geometry x = rows_of(input), y = rows_of(output);
        DISTCONV_CHECK_H2X(h2x_layer_norm_forward(Tensor::h2x_type(), Tensor::h2x_type(), num_rows(x), channels(x), &x, &y,
                                                  input.get_const_base_ptr(), scale, bias, output.get_base_ptr(), mean, rstd,
                                                  m_epsilon, m_stream));
        return 0;
    }

    // The weights' gradients are overwritten; either may be nullptr.
    template <typename Tensor>
    int backward(const Tensor& input, const Tensor& d_output, const typename Tensor::data_type* mean,
                 const typename Tensor::data_type* rstd, const typename Tensor::data_type* scale, Tensor& d_input,
                 typename Tensor::data_type* d_scale, typename Tensor::data_type* d_bias)
    {
        const h2x_tensor_geometry x = rows_of(input), dy = rows_of(d_output), dx = rows_of(d_input);
        const h2x_dtype type = Tensor::h2x_type();
        void* const workspace = m_workspace.get(d_scale || d_bias ? h2x_layer_norm_workspace_bytes(type, num_rows(x), channels(x)) : 0);
        DISTCONV_CHECK_H2X(h2x_layer_norm_backward(type, type, num_rows(x), channels(x), &x, &dy, &dx, input.get_const_base_ptr(),
                                                   d_output.get_const_base_ptr(), mean, rstd, scale, d_input.get_base_ptr(),
                                                   d_scale, d_bias, workspace, m_stream));
        return 0;
    }

private:
    template <typename Tensor>
    static h2x_tensor_geometry rows_of(const Tensor& t)
    {
        h2x_tensor_geometry g = {};
        g.num_dims = t.get_num_dims();
        const auto strides = t.get_strides();
        for (int i = 0; i < g.num_dims; ++i)
        {
            g.local_shape[i] = static_cast<int64_t>(t.get_local_shape()[i]);
            g.strides[i] = static_cast<int64_t>(strides[i]);
        }
        return g;
    }
    static int channels(const h2x_tensor_geometry& g) { return static_cast<int>(g.local_shape[0]); }
    static size_t num_rows(const h2x_tensor_geometry& g)
    {
        size_t n = 1;
        for (int i = 1; i < g.num_dims; ++i)
            n *= static_cast<size_t>(g.local_shape[i]);
        return n;
    }

    hipStream_t m_stream;
    double m_epsilon;
    TokenWorkspace m_workspace;
};

template <typename Backend>
class RotaryPositions;

// Pair i of an axis with m pairs turns by position * base^(-i / m).
template <>
class RotaryPositions<BackendMI355X>
{
public:
    RotaryPositions(BackendMI355X const& backend, const std::vector<int>& axis_pairs, double base = 10000.0,
                    h2x_rotary_pairing pairing = H2X_ROTARY_HALVES)
        : m_stream(backend.get_stream()), m_axis_pairs(axis_pairs), m_pairing(pairing)
    {
        assert_always(axis_pairs.size() <= H2X_MAX_AXES);
        std::vector<double> frequencies;
        for (const int m : axis_pairs)
            for (int i = 0; i < m; ++i)
                frequencies.push_back(std::pow(base, -static_cast<double>(i) / m));
        m_frequencies.allocate(frequencies.size() * sizeof(double) + 1);
        DISTCONV_CHECK_HIP(hipMemcpy(m_frequencies.get(), frequencies.data(), frequencies.size() * sizeof(double),
                                     hipMemcpyHostToDevice));
    }

    // heads: type, sizes and strides of x and y, and the positions' strides; the axes and the pairing are the layer's.
    int forward(h2x_rotary heads, const void* x, const int32_t* positions, void* y) { return apply(heads, x, positions, 0, y); }
    int backward(h2x_rotary heads, const void* dy, const int32_t* positions, void* dx)
    {
        return apply(heads, dy, positions, 1, dx);
    }

private:
    int apply(h2x_rotary& heads, const void* x, const int32_t* positions, int inverse, void* y)
    {
        heads.pairing = m_pairing;
        heads.num_axes = static_cast<int32_t>(m_axis_pairs.size());
        for (size_t i = 0; i < m_axis_pairs.size(); ++i)
            heads.axis_pairs[i] = m_axis_pairs[i];
        DISTCONV_CHECK_H2X(h2x_rotary_apply(&heads, x, positions, static_cast<const double*>(m_frequencies.get()), inverse, y,
                                            m_stream));
        return 0;
    }

    hipStream_t m_stream;
    std::vector<int> m_axis_pairs;
    h2x_rotary_pairing m_pairing;
    tensor::Memory<tensor::CUDAAllocator> m_frequencies;
};

template <typename Backend>
class Attention;

template <>
class Attention<BackendMI355X>
{
public:
    explicit Attention(BackendMI355X const& backend) : m_stream(backend.get_stream()) {}

    int forward(const h2x_attention& a, const void* q, const void* k, const void* v, void* o, float* logsumexp = nullptr,
                const int32_t* query_lengths = nullptr, const int32_t* key_lengths = nullptr)
    {
        DISTCONV_CHECK_H2X(h2x_attention_forward(&a, q, k, v, query_lengths, key_lengths, o, logsumexp,
                                                 m_workspace.get(h2x_attention_forward_workspace_bytes(&a)), m_stream));
        return 0;
    }

    int backward(const h2x_attention& a, const void* q, const void* k, const void* v, const void* o, const void* d_o,
                 const float* logsumexp, void* dq, void* dk, void* dv, const int32_t* query_lengths = nullptr,
                 const int32_t* key_lengths = nullptr)
    {
        DISTCONV_CHECK_H2X(h2x_attention_backward(&a, q, k, v, o, d_o, logsumexp, query_lengths, key_lengths, dq, dk, dv,
                                                  m_workspace.get(h2x_attention_backward_workspace_bytes(&a)), m_stream));
        return 0;
    }

private:
    hipStream_t m_stream;
    TokenWorkspace m_workspace;
};

} // namespace distconv
