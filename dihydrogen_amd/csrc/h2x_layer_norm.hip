// Layer normalisation of rows, forward and backward (include/h2x.h has the formulas).
//
// Both directions are bound by memory: forward reads x and writes y, backward reads x and dy and writes dx, once each.
// A row is held in registers from its only read to its write, so that the variance can be summed about the mean (two
// passes over registers) without a second read.  A row belongs to a wave where it fits, which then needs neither LDS nor
// barriers; longer ones to a workgroup; rows beyond what a workgroup holds are read again (they come from L2).
#include "h2x_token.hpp"

namespace h2x
{
namespace token
{
namespace
{

template <typename T>
constexpr int kVec = 16 / sizeof(T); // elements of a 16-byte load

// Threads of a row, and how many 16-byte vectors of it each thread holds.
template <int Threads, int Vectors>
struct Shape
{
    static constexpr int threads = Threads, vectors = Vectors;
};

// Sum over the Threads of a row; all of them get it.  lds: one place a wave, of which two sets alternate between sums, so
// that a barrier a sum is enough.
template <int Threads, typename W>
__device__ __forceinline__ W row_total(W v, W* lds)
{
    v = wave_total(v);
    if constexpr (Threads > kWaveSize)
    {
        if ((threadIdx.x & (kWaveSize - 1)) == 0)
            lds[threadIdx.x / kWaveSize] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < Threads / kWaveSize; ++w)
            v += lds[w];
    }
    return v;
}

// Elements at .. at + V - 1 of a row of c elements that begins anywhere; what lies behind its end is `rest`.
template <typename T, typename W, int V>
__device__ __forceinline__ void load(const T* row, int at, int c, W (&v)[V], W rest)
{
    if (at + V <= c)
    {
        const UVec<T, V> x = *reinterpret_cast<const UVec<T, V>*>(row + at);
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[i] = static_cast<W>(x.v[i]);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[i] = at + i < c ? static_cast<W>(row[at + i]) : rest;
    }
}
template <typename T, typename W, int V>
__device__ __forceinline__ void store(T* row, int at, int c, const W (&v)[V])
{
    if (at + V <= c)
    {
        UVec<T, V> x;
#pragma unroll
        for (int i = 0; i < V; ++i)
            x.v[i] = static_cast<T>(v[i]);
        *reinterpret_cast<UVec<T, V>*>(row + at) = x;
    }
    else
    {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (at + i < c)
                row[at + i] = static_cast<T>(v[i]);
    }
}

template <typename W>
__device__ __forceinline__ W fma_(W a, W b, W c)
{
    if constexpr (sizeof(W) == 8)
        return __builtin_fma(a, b, c);
    else
        return __builtin_fmaf(a, b, c);
}
template <typename W>
__device__ __forceinline__ W reciprocal_root(W v)
{
    return W(1) / (sizeof(W) == 8 ? sqrt(v) : sqrtf(v));
}

template <typename T, typename P>
struct Forward
{
    const T* x;
    const P *scale, *bias;
    T* y;
    wide<T>*mean, *rstd;
    Rows x_rows, y_rows;
    uint32_t first, num_rows; // rows of the launch begin at `first`
    int channels;
    wide<T> epsilon;
};

// Rows in registers.  A workgroup of Threads threads a row, or (Threads = 64) of any number of waves with a row each.
template <typename T, typename P, typename S>
__global__ void __launch_bounds__(S::threads == 64 ? 256 : S::threads) ln_forward_kernel(const Forward<T, P> a)
{
    using W = wide<T>;
    constexpr int V = kVec<T>, K = S::vectors;
    constexpr bool kWaveRows = S::threads == kWaveSize;
    __shared__ W lds[2][S::threads / kWaveSize];
    const uint32_t wave = threadIdx.x / kWaveSize;
    const uint32_t r = a.first + (kWaveRows ? blockIdx.x * (blockDim.x / kWaveSize) + wave : blockIdx.x);
    const int t = kWaveRows ? threadIdx.x & (kWaveSize - 1) : threadIdx.x;
    if (r >= a.num_rows)
        return;
    const int c = a.channels;
    const T* const x = a.x + row_offset(a.x_rows, r);
    T* const y = a.y + row_offset(a.y_rows, r);
    W v[K][V], sum = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
        load(x, (k * S::threads + t) * V, c, v[k], W(0));
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
            sum += v[k][i];
    const W mean = row_total<S::threads>(sum, lds[0]) / c;
    W squares = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
            const W d = (k * S::threads + t) * V + i < c ? v[k][i] - mean : W(0);
            squares = fma_(d, d, squares);
        }
    const W rstd = reciprocal_root(row_total<S::threads>(squares, lds[1]) / c + a.epsilon);
    if (a.mean && t == 0)
    {
        a.mean[r] = mean;
        a.rstd[r] = rstd;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
    {
        const int at = (k * S::threads + t) * V;
        if (at >= c)
            continue;
        W w[V], b[V];
#pragma unroll
        for (int i = 0; i < V; ++i)
            w[i] = W(1), b[i] = W(0);
        if (a.scale)
            load(a.scale, at, c, w, W(1));
        if (a.bias)
            load(a.bias, at, c, b, W(0));
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[k][i] = fma_((v[k][i] - mean) * rstd, w[i], b[i]);
        store(y, at, c, v[k]);
    }
}

// Rows beyond the registers of a workgroup: three passes over a row, the second and third out of L2.  Threads keep partial sums
// in 64 bits.
constexpr int kLongThreads = 1024;
template <typename T, typename P>
__global__ void __launch_bounds__(kLongThreads) ln_forward_long_kernel(const Forward<T, P> a)
{
    using W = wide<T>;
    constexpr int V = kVec<T>;
    __shared__ double lds[2][kLongThreads / kWaveSize];
    const int c = a.channels, t = threadIdx.x;
    const uint32_t r = a.first + blockIdx.x;
    const T* const x = a.x + row_offset(a.x_rows, r);
    T* const y = a.y + row_offset(a.y_rows, r);
    double sum = 0, squares = 0;
    for (int64_t at = t * V; at < c; at += kLongThreads * V)
    {
        W v[V], part = 0;
        load(x, static_cast<int>(at), c, v, W(0));
#pragma unroll
        for (int i = 0; i < V; ++i)
            part += v[i];
        sum += part;
    }
    const W mean = static_cast<W>(row_total<kLongThreads>(sum, lds[0]) / c);
    for (int64_t at = t * V; at < c; at += kLongThreads * V)
    {
        W v[V], part = 0;
        load(x, static_cast<int>(at), c, v, mean);
#pragma unroll
        for (int i = 0; i < V; ++i)
            part = fma_(v[i] - mean, v[i] - mean, part);
        squares += part;
    }
    const W rstd = reciprocal_root(static_cast<W>(row_total<kLongThreads>(squares, lds[1]) / c) + a.epsilon);
    if (a.mean && t == 0)
    {
        a.mean[r] = mean;
        a.rstd[r] = rstd;
    }
    for (int64_t at = t * V; at < c; at += kLongThreads * V)
    {
        W v[V], w[V], b[V];
        load(x, static_cast<int>(at), c, v, W(0));
#pragma unroll
        for (int i = 0; i < V; ++i)
            w[i] = W(1), b[i] = W(0);
        if (a.scale)
            load(a.scale, static_cast<int>(at), c, w, W(1));
        if (a.bias)
            load(a.bias, static_cast<int>(at), c, b, W(0));
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[i] = fma_((v[i] - mean) * rstd, w[i], b[i]);
        store(y, static_cast<int>(at), c, v);
    }
}

template <typename T, typename P>
struct Backward
{
    const T *x, *dy;
    const wide<T>*mean, *rstd;
    const P* scale;
    T* dx;             // or NULL
    wide<T>* partials; // [2][workgroups][channels]: sums of dy * h and of dy over a workgroup's rows; or NULL
    Rows x_rows, dy_rows, dx_rows;
    uint32_t first, num_rows; // (long rows: those of the launch begin at `first`)
    int channels;
};

// Row r, x and dy of which thread t holds: dx to memory, what the row adds to the weights' gradients to dscale and dbias.
template <typename T, typename P, typename S, bool Weights, int K, int V>
__device__ __forceinline__ void ln_backward_row(const Backward<T, P>& a, uint32_t r, int t, wide<T> (*lds)[16],
                                                wide<T> (&dscale)[K][V], wide<T> (&dbias)[K][V])
{
    using W = wide<T>;
    const int c = a.channels;
    const T* const x = a.x + row_offset(a.x_rows, r);
    const T* const dy = a.dy + row_offset(a.dy_rows, r);
    const W mean = a.mean[r], rstd = a.rstd[r];
    W h[K][V], g[K][V], sum = 0, dot = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
    {
        const int at = (k * S::threads + t) * V;
        load(x, at, c, h[k], mean);
        load(dy, at, c, g[k], W(0));
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
    {
        const int at = (k * S::threads + t) * V;
        W w[V];
#pragma unroll
        for (int i = 0; i < V; ++i)
            w[i] = W(1);
        if (a.scale && at < c)
            load(a.scale, at, c, w, W(0));
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
            h[k][i] = (h[k][i] - mean) * rstd;
            if constexpr (Weights)
            {
                dscale[k][i] = fma_(g[k][i], h[k][i], dscale[k][i]);
                dbias[k][i] += g[k][i];
            }
            g[k][i] *= w[i];
            sum += g[k][i];
            dot = fma_(g[k][i], h[k][i], dot);
        }
    }
    if (!a.dx)
        return;
    sum = row_total<S::threads>(sum, lds[0]) / c;
    dot = row_total<S::threads>(dot, lds[1]) / c;
    T* const dx = a.dx + row_offset(a.dx_rows, r);
#pragma unroll
    for (int k = 0; k < K; ++k)
    {
        const int at = (k * S::threads + t) * V;
        if (at >= c)
            continue;
#pragma unroll
        for (int i = 0; i < V; ++i)
            g[k][i] = rstd * (g[k][i] - fma_(h[k][i], dot, sum));
        store(dx, at, c, g[k]);
    }
}

// Rows in registers.  A workgroup goes through every gridDim.x-th row (of its waves each, where rows belong to waves) and keeps
// the sums for the weights' gradients in registers, a column a place; its waves' sums meet in LDS at the end, in the waves' order.
template <typename T, typename P, typename S, bool Weights>
__global__ void __launch_bounds__(S::threads == 64 ? 256 : S::threads) ln_backward_kernel(const Backward<T, P> a)
{
    using W = wide<T>;
    constexpr int V = kVec<T>, K = S::vectors;
    constexpr bool kWaveRows = S::threads == kWaveSize;
    constexpr int kWaves = kWaveRows ? 4 : 1; // with rows of their own
    __shared__ W lds[2][2][16];
    const int wave = threadIdx.x / kWaveSize;
    const int t = kWaveRows ? threadIdx.x & (kWaveSize - 1) : threadIdx.x;
    W dscale[K][V], dbias[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
            dscale[k][i] = dbias[k][i] = W(0);
    // (all threads of a workgroup whose rows are its own go round equally often)
    int turn = 0;
    for (uint64_t r = kWaveRows ? blockIdx.x * kWaves + wave : blockIdx.x; r < a.num_rows;
         r += static_cast<uint64_t>(gridDim.x) * kWaves)
        ln_backward_row<T, P, S, Weights>(a, static_cast<uint32_t>(r), t, lds[turn ^= 1], dscale, dbias);
    if constexpr (Weights)
    {
        const int c = a.channels;
        W* const out = a.partials + static_cast<size_t>(blockIdx.x) * c;
        const size_t half = static_cast<size_t>(gridDim.x) * c;
        if constexpr (kWaveRows)
        {
            __shared__ W sums[kWaves - 1][kWaveSize * V];
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int which = 0; which < 2; ++which)
                {
                    W(&mine)[V] = which ? dbias[k] : dscale[k];
                    __syncthreads();
                    if (wave > 0)
                    {
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            sums[wave - 1][i * kWaveSize + t] = mine[i];
                    }
                    __syncthreads();
                    const int at = (k * kWaveSize + t) * V;
                    if (wave == 0 && at < c)
                    {
#pragma unroll
                        for (int i = 0; i < V; ++i)
#pragma unroll
                            for (int w = 0; w < kWaves - 1; ++w)
                                mine[i] += sums[w][i * kWaveSize + t];
                        store(out + which * half, at, c, mine);
                    }
                }
        }
        else
        {
#pragma unroll
            for (int k = 0; k < K; ++k)
            {
                const int at = (k * S::threads + t) * V;
                if (at < c)
                {
                    store(out, at, c, dscale[k]);
                    store(out + half, at, c, dbias[k]);
                }
            }
        }
    }
}

// Rows beyond the registers of a workgroup: dx in two passes over a row.
template <typename T, typename P>
__global__ void __launch_bounds__(kLongThreads) ln_backward_long_kernel(const Backward<T, P> a)
{
    using W = wide<T>;
    constexpr int V = kVec<T>;
    __shared__ double lds[2][kLongThreads / kWaveSize];
    const int c = a.channels, t = threadIdx.x;
    const uint32_t r = a.first + blockIdx.x;
    const T* const x = a.x + row_offset(a.x_rows, r);
    const T* const dy = a.dy + row_offset(a.dy_rows, r);
    T* const dx = a.dx + row_offset(a.dx_rows, r);
    const W mean = a.mean[r], rstd = a.rstd[r];
    double sums = 0, dots = 0;
    W sum = 0, dot = 0;
    for (int pass = 0; pass < 2; ++pass)
    {
        for (int64_t at = t * V; at < c; at += kLongThreads * V)
        {
            W h[V], g[V], w[V], s = 0, d = 0;
            load(x, static_cast<int>(at), c, h, mean);
            load(dy, static_cast<int>(at), c, g, W(0));
#pragma unroll
            for (int i = 0; i < V; ++i)
                w[i] = W(1);
            if (a.scale)
                load(a.scale, static_cast<int>(at), c, w, W(0));
#pragma unroll
            for (int i = 0; i < V; ++i)
            {
                h[i] = (h[i] - mean) * rstd;
                g[i] *= w[i];
                s += g[i];
                d = fma_(g[i], h[i], d);
                g[i] = rstd * (g[i] - fma_(h[i], dot, sum));
            }
            sums += s;
            dots += d;
            if (pass == 1)
                store(dx, static_cast<int>(at), c, g);
        }
        if (pass == 0)
        {
            sum = static_cast<W>(row_total<kLongThreads>(sums, lds[0]) / c);
            dot = static_cast<W>(row_total<kLongThreads>(dots, lds[1]) / c);
        }
    }
}

// Their weights' gradients: a workgroup takes 256 vectors of columns and every gridDim.y-th row.
template <typename T, typename P>
__global__ void __launch_bounds__(kBlockSize) ln_weights_long_kernel(const Backward<T, P> a)
{
    using W = wide<T>;
    constexpr int V = kVec<T>;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * kBlockSize + threadIdx.x) * V;
    const int c = a.channels;
    if (first >= c)
        return;
    const int at = static_cast<int>(first);
    W dscale[V], dbias[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
        dscale[i] = dbias[i] = W(0);
    for (uint64_t r = blockIdx.y; r < a.num_rows; r += gridDim.y)
    {
        const W mean = a.mean[r], rstd = a.rstd[r];
        W h[V], g[V];
        load(a.x + row_offset(a.x_rows, static_cast<uint32_t>(r)), at, c, h, mean);
        load(a.dy + row_offset(a.dy_rows, static_cast<uint32_t>(r)), at, c, g, W(0));
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
            dscale[i] = fma_(g[i], (h[i] - mean) * rstd, dscale[i]);
            dbias[i] += g[i];
        }
    }
    W* const out = a.partials + static_cast<size_t>(blockIdx.y) * c;
    store(out, at, c, dscale);
    store(out + static_cast<size_t>(gridDim.y) * c, at, c, dbias);
}

// Sums over the workgroups' partials, in 64 bits: 16 columns by 64 lanes of rows a workgroup, the lanes' sums in order.
constexpr int kSumColumns = 16, kSumLanes = 64;
template <typename W, typename P>
__global__ void __launch_bounds__(kSumColumns* kSumLanes)
    ln_weights_sum_kernel(const W* partials, int parts, int channels, P* dscale, P* dbias)
{
    __shared__ double lds[kSumLanes][kSumColumns + 1];
    const int column = threadIdx.x % kSumColumns, lane = threadIdx.x / kSumColumns;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kSumColumns + column;
    P* const out = blockIdx.y ? dbias : dscale;
    if (!out)
        return;
    double sum = 0;
    if (c < channels)
    {
        const W* p = partials + static_cast<size_t>(blockIdx.y) * parts * channels + c;
        for (int i = lane; i < parts; i += kSumLanes)
            sum += p[static_cast<size_t>(i) * channels];
    }
    lds[lane][column] = sum;
#pragma unroll
    for (int n = kSumLanes / 2; n >= 1; n /= 2)
    {
        __syncthreads();
        if (lane < n)
            lds[lane][column] += lds[lane + n][column];
    }
    if (lane == 0 && c < channels)
        out[c] = static_cast<P>(static_cast<wide<P>>(lds[0][column]));
}

// ---- host ----------------------------------------------------------------------

// Elements of a row that fit the registers of one wave, 256 and 1024 threads with so many vectors a thread.
constexpr int kMostVectors = 4;

// How the rows are shared out.
struct Split
{
    int threads, vectors; // of a row; threads = 0: too long for registers
};
Split split_rows(int vec, int channels)
{
    const int64_t vectors = (static_cast<int64_t>(channels) + vec - 1) / vec;
    for (const int threads : {64, 256, 1024})
        for (int k = 1; k <= (threads == 1024 ? 2 : kMostVectors); k *= 2)
            if (vectors <= static_cast<int64_t>(threads) * k)
                return {threads, k};
    return {0, 0};
}

// Workgroups whose sums for the weights' gradients are added up at the end: two for each CU where rows are that many.
uint32_t weight_parts(int threads, size_t num_rows)
{
    const size_t rows_at_once = threads == 64 ? 4 : 1;
    const size_t most = 2 * 256, groups = (num_rows + rows_at_once - 1) / rows_at_once;
    return static_cast<uint32_t>(groups < most ? (groups ? groups : 1) : most);
}

template <typename F>
int with_shape(const Split& s, const F& f)
{
    const auto by_vectors = [&](auto threads) {
        constexpr int N = decltype(threads)::value;
        return s.vectors == 1   ? f(Shape<N, 1>())
               : s.vectors == 2 ? f(Shape<N, 2>())
                                : f(Shape<N, 4>());
    };
    return s.threads == 64    ? by_vectors(std::integral_constant<int, 64>())
           : s.threads == 256 ? by_vectors(std::integral_constant<int, 256>())
                              : by_vectors(std::integral_constant<int, 1024>());
}

// f(workgroups) for as many launches as a grid of fewer than 2^32 threads makes necessary, a.first set for each.
template <typename A, typename F>
void each_launch(A* a, uint32_t rows_each, uint32_t threads, const F& f)
{
    const uint32_t most = 0x80000000u / threads;
    const uint64_t groups = (static_cast<uint64_t>(a->num_rows) + rows_each - 1) / rows_each;
    for (uint64_t g = 0; g < groups; g += most)
    {
        a->first = static_cast<uint32_t>(g * rows_each);
        f(dim3(static_cast<uint32_t>(groups - g < most ? groups - g : most)));
    }
}

template <typename T, typename P>
int forward(Forward<T, P> a, hipStream_t stream)
{
    const Split s = split_rows(kVec<T>, a.channels);
    if (s.threads == 0)
    {
        each_launch(&a, 1, kLongThreads, [&](dim3 grid) {
            launch(ln_forward_long_kernel<T, P>, grid, dim3(kLongThreads), stream, a);
        });
        return launch_status();
    }
    return with_shape(s, [&](auto shape) {
        using S = decltype(shape);
        // a wave's rows: four waves a workgroup, one where rows are fewer than the waves that run at once
        const uint32_t waves = S::threads > 64 || a.num_rows <= 4 * chip_units() ? 1 : 4;
        each_launch(&a, waves, S::threads * waves, [&](dim3 grid) {
            launch(ln_forward_kernel<T, P, S>, grid, dim3(S::threads * waves), stream, a);
        });
        return launch_status();
    });
}

template <typename T, typename P>
int backward(Backward<T, P> a, P* dscale, P* dbias, hipStream_t stream)
{
    const Split s = split_rows(kVec<T>, a.channels);
    const bool weights = dscale || dbias;
    const uint32_t parts = weight_parts(s.threads, a.num_rows);
    if (s.threads == 0)
    {
        if (weights) // first: dx may lie where x or dy does
        {
            const int64_t vectors = (static_cast<int64_t>(a.channels) + kVec<T> - 1) / kVec<T>;
            launch(ln_weights_long_kernel<T, P>, dim3(static_cast<uint32_t>((vectors + kBlockSize - 1) / kBlockSize), parts),
                   dim3(kBlockSize), stream, a);
        }
        if (a.dx)
            each_launch(&a, 1, kLongThreads, [&](dim3 grid) {
                launch(ln_backward_long_kernel<T, P>, grid, dim3(kLongThreads), stream, a);
            });
    }
    else
    {
        (void) with_shape(s, [&](auto shape) {
            using S = decltype(shape);
            constexpr uint32_t kThreads = S::threads == 64 ? 256 : S::threads;
            constexpr uint32_t kRows = S::threads == 64 ? 4 : 1, kMost = 0x80000000u / kThreads;
            const uint32_t groups = (a.num_rows + kRows - 1) / kRows;
            if (weights)
                launch(ln_backward_kernel<T, P, S, true>, dim3(parts), dim3(kThreads), stream, a);
            else
                launch(ln_backward_kernel<T, P, S, false>, dim3(groups < kMost ? groups : kMost), dim3(kThreads), stream, a);
            return 0;
        });
    }
    if (weights)
        launch(ln_weights_sum_kernel<wide<T>, P>, dim3((a.channels + kSumColumns - 1) / kSumColumns, 2),
               dim3(kSumColumns * kSumLanes), stream, a.partials, static_cast<int>(parts), a.channels, dscale, dbias);
    return launch_status();
}

// f(T(), P()) for the types of the elements and of the weights.
template <typename F>
int with_types(int dtype, int weight_dtype, const F& f)
{
    switch (dtype)
    {
    case H2X_F32: return weight_dtype == H2X_F32 ? f(float(), float()) : H2X_ERR_UNSUPPORTED;
    case H2X_F64: return weight_dtype == H2X_F64 ? f(double(), double()) : H2X_ERR_UNSUPPORTED;
    case H2X_BF16:
        return weight_dtype == H2X_F32    ? f(bf16(), float())
               : weight_dtype == H2X_BF16 ? f(bf16(), bf16())
                                          : H2X_ERR_UNSUPPORTED;
    case H2X_F16:
        return weight_dtype == H2X_F32   ? f(f16(), float())
               : weight_dtype == H2X_F16 ? f(f16(), f16())
                                         : H2X_ERR_UNSUPPORTED;
    default: return H2X_ERR_UNSUPPORTED;
    }
}

} // namespace
} // namespace token
} // namespace h2x

using namespace h2x;
using namespace h2x::token;

extern "C" int h2x_layer_norm_forward(h2x_dtype dtype, h2x_dtype weight_dtype, size_t num_rows, int num_channels,
                                      const h2x_tensor_geometry* x_rows, const h2x_tensor_geometry* y_rows, const void* x,
                                      const void* scale, const void* bias, void* y, void* mean, void* rstd, double epsilon,
                                      h2x_stream_t stream)
{
    return with_types(dtype, weight_dtype, [&](auto t, auto p) -> int {
        using T = decltype(t);
        using P = decltype(p);
        if (num_channels < 1 || !(epsilon >= 0) || (mean == nullptr) != (rstd == nullptr))
            return H2X_ERR_INVALID_ARGUMENT;
        if (num_rows > 0x7fffffffu)
            return H2X_ERR_TOO_LARGE;
        Forward<T, P> a{static_cast<const T*>(x), static_cast<const P*>(scale), static_cast<const P*>(bias),
                        static_cast<T*>(y),       static_cast<wide<T>*>(mean),  static_cast<wide<T>*>(rstd)};
        if (!make_rows(x_rows, num_rows, num_channels, &a.x_rows) || !make_rows(y_rows, num_rows, num_channels, &a.y_rows))
            return H2X_ERR_INVALID_ARGUMENT;
        if (num_rows == 0)
            return H2X_SUCCESS;
        if (!x || !y)
            return H2X_ERR_INVALID_ARGUMENT;
        a.num_rows = static_cast<uint32_t>(num_rows);
        a.channels = num_channels;
        a.epsilon = static_cast<wide<T>>(epsilon);
        return forward(a, as_stream(stream));
    });
}

extern "C" size_t h2x_layer_norm_workspace_bytes(h2x_dtype dtype, size_t num_rows, int num_channels)
{
    const int size = element_size(dtype);
    if (size == 0 || num_channels < 1)
        return 0;
    const uint32_t parts = weight_parts(split_rows(16 / size, num_channels).threads, num_rows);
    return 2 * static_cast<size_t>(parts) * num_channels * (size == 8 ? 8 : 4);
}

extern "C" int h2x_layer_norm_backward(h2x_dtype dtype, h2x_dtype weight_dtype, size_t num_rows, int num_channels,
                                       const h2x_tensor_geometry* x_rows, const h2x_tensor_geometry* dy_rows,
                                       const h2x_tensor_geometry* dx_rows, const void* x, const void* dy, const void* mean,
                                       const void* rstd, const void* scale, void* dx, void* dscale, void* dbias,
                                       void* workspace, h2x_stream_t stream)
{
    return with_types(dtype, weight_dtype, [&](auto t, auto p) -> int {
        using T = decltype(t);
        using P = decltype(p);
        if (num_channels < 1)
            return H2X_ERR_INVALID_ARGUMENT;
        if (num_rows > 0x7fffffffu)
            return H2X_ERR_TOO_LARGE;
        const bool weights = dscale || dbias;
        Backward<T, P> a{static_cast<const T*>(x),          static_cast<const T*>(dy),
                         static_cast<const wide<T>*>(mean), static_cast<const wide<T>*>(rstd),
                         static_cast<const P*>(scale),      static_cast<T*>(dx),
                         static_cast<wide<T>*>(workspace)};
        if (!make_rows(x_rows, num_rows, num_channels, &a.x_rows) || !make_rows(dy_rows, num_rows, num_channels, &a.dy_rows)
            || !make_rows(dx_rows, num_rows, num_channels, &a.dx_rows))
            return H2X_ERR_INVALID_ARGUMENT;
        if ((weights && !workspace) || (num_rows > 0 && (!x || !dy || !mean || !rstd)))
            return H2X_ERR_INVALID_ARGUMENT;
        if (!weights && (!dx || num_rows == 0))
            return H2X_SUCCESS;
        a.num_rows = static_cast<uint32_t>(num_rows);
        a.channels = num_channels;
        return backward(a, static_cast<P*>(dscale), static_cast<P*>(dbias), as_stream(stream));
    });
}
