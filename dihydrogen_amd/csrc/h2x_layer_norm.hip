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
    static constexpr bool wave_rows = Threads <= kWaveSize; // a workgroup's waves have rows of their own, one or several at a time
    static constexpr int rows_of_wave = wave_rows ? kWaveSize / Threads : 1;
    static constexpr int most_threads = wave_rows ? kBlockSize : Threads;
};

// Sum over each G lanes of a wave, a power of two from 8 on; all of them get it.
template <int G, typename W>
__device__ __forceinline__ W group_total(W v)
{
    constexpr int kHalfMirror = 0x141; // lane i of eight and lane 7 - i
    const auto add = [](W a, W b) { return a + b; };
    if constexpr (G == 64)
        return wave_total(v);
    if constexpr (G == 32)
        v = combine_apart<16>(v, add);
    if constexpr (G >= 16)
    {
        v += dpp_move<kDppRowRor8>(v);
        v += dpp_move<kDppRowRor4>(v); // lanes 8 apart hold the same
    }
    else
        v += dpp_move<kHalfMirror>(v);
    v += dpp_move<kDppQuadSwap2>(v);
    return v + dpp_move<kDppQuadSwap1>(v);
}

// Sum over the Threads of a row; all of them get it.  lds: one place a wave, of which two sets alternate between sums, so
// that a barrier a sum is enough.
template <int Threads, typename W>
__device__ __forceinline__ W row_total(W v, W* lds)
{
    v = group_total<(Threads < kWaveSize ? Threads : kWaveSize)>(v);
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

// Elements at .. at + V - 1 of a row of c elements that begins anywhere; zero behind its end.
template <int V, typename T>
__device__ __forceinline__ UVec<T, V> load(const T* row, int at, int c)
{
    UVec<T, V> x;
    if (at + V <= c)
        x = *reinterpret_cast<const UVec<T, V>*>(row + at);
    else
    {
#pragma unroll
        for (int i = 0; i < V; ++i)
            x.v[i] = at + i < c ? row[at + i] : static_cast<T>(0.0f);
    }
    return x;
}
// A thread's vectors of a row.
template <typename S, int V, typename T>
__device__ __forceinline__ void load_row(const T* row, int t, int c, UVec<T, V> (&x)[S::vectors])
{
#pragma unroll
    for (int k = 0; k < S::vectors; ++k)
        x[k] = load<V>(row, (k * S::threads + t) * V, c);
}
// Its weights; `none` where there are none.
template <typename S, int V, typename P>
__device__ __forceinline__ void load_weights(const P* weights, float none, int t, int c, UVec<P, V> (&x)[S::vectors])
{
    if (weights)
        load_row<S, V>(weights, t, c, x);
    else
    {
#pragma unroll
        for (int k = 0; k < S::vectors; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
                x[k].v[i] = static_cast<P>(none);
    }
}
// streamed: past the caches.
template <typename T, typename W, int V>
__device__ __forceinline__ void store(T* row, int at, int c, const W (&v)[V], bool streamed = false)
{
    if (at + V <= c)
    {
        typedef unsigned int Words __attribute__((ext_vector_type(sizeof(T) * V / 4), aligned(sizeof(T))));
        UVec<T, V> x;
#pragma unroll
        for (int i = 0; i < V; ++i)
            x.v[i] = static_cast<T>(v[i]);
        if (streamed)
            __builtin_nontemporal_store(__builtin_bit_cast(Words, x), reinterpret_cast<Words*>(row + at));
        else
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
    uint32_t num_rows;
    int channels;
    wide<T> epsilon;
    bool streamed; // y
};

// Rows in registers.  A workgroup (of waves with a row each, or of one row) goes through every gridDim.x-th of them; scale and bias stay in
// registers, and the next row is on its way while one is worked on, where that leaves registers.  (32768 x 1024 in bf16 with a
// workgroup for each four rows: 35 us, 3.8 TB/s.)
template <typename T, typename P, typename S>
__global__ void __launch_bounds__(S::most_threads) ln_forward_kernel(const Forward<T, P> a)
{
    using W = wide<T>;
    constexpr int V = kVec<T>, K = S::vectors;
    constexpr bool kAhead = K * V <= 16;
    __shared__ W lds[2][2][S::wave_rows ? 1 : S::threads / kWaveSize];
    const uint32_t at_once = S::wave_rows ? blockDim.x / S::threads : 1; // rows
    const uint32_t step = gridDim.x * at_once;
    uint32_t r = blockIdx.x * at_once + (S::wave_rows ? threadIdx.x / S::threads : 0);
    const int t = threadIdx.x % S::threads, c = a.channels;
    if (r >= a.num_rows)
        return;
    UVec<T, V> x[K], next[kAhead ? K : 1];
    UVec<P, V> w[K], b[K];
    load_row<S, V>(a.x + row_offset(a.x_rows, r), t, c, x);
    load_weights<S, V>(a.scale, 1.0f, t, c, w);
    load_weights<S, V>(a.bias, 0.0f, t, c, b);
    for (int turn = 0;; turn ^= 1)
    {
        const uint32_t following = r + step;
        const bool more = following < a.num_rows;
        if constexpr (kAhead)
        {
            if (more)
                load_row<S, V>(a.x + row_offset(a.x_rows, following), t, c, next);
        }
        W v[K][V], sum = 0;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
            {
                v[k][i] = static_cast<W>(x[k].v[i]);
                sum += v[k][i];
            }
        const W mean = row_total<S::threads>(sum, lds[turn][0]) / c;
        W squares = 0;
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            const int at = (k * S::threads + t) * V;
#pragma unroll
            for (int i = 0; i < V; ++i)
                v[k][i] -= mean;
            if (at + V > c)
            {
                // what lies behind the row's end counts nothing
#pragma unroll
                for (int i = 0; i < V; ++i)
                    v[k][i] = at + i < c ? v[k][i] : W(0);
            }
#pragma unroll
            for (int i = 0; i < V; ++i)
                squares = fma_(v[k][i], v[k][i], squares);
        }
        const W rstd = reciprocal_root(row_total<S::threads>(squares, lds[turn][1]) / c + a.epsilon);
        if (a.mean && t == 0)
        {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        T* const y = a.y + row_offset(a.y_rows, r);
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            const int at = (k * S::threads + t) * V;
            if (at >= c)
                continue;
#pragma unroll
            for (int i = 0; i < V; ++i)
                v[k][i] = fma_(v[k][i] * rstd, static_cast<W>(w[k].v[i]), static_cast<W>(b[k].v[i]));
            store(y, at, c, v[k], a.streamed);
        }
        if (!more)
            return;
        r = following;
        if constexpr (kAhead)
        {
#pragma unroll
            for (int k = 0; k < K; ++k)
                x[k] = next[k];
        }
        else
            load_row<S, V>(a.x + row_offset(a.x_rows, r), t, c, x);
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
    for (uint32_t r = blockIdx.x; r < a.num_rows; r += gridDim.x)
    {
        const T* const x = a.x + row_offset(a.x_rows, r);
        T* const y = a.y + row_offset(a.y_rows, r);
        double sum = 0, squares = 0;
        for (int64_t at = t * V; at < c; at += kLongThreads * V)
        {
            const UVec<T, V> v = load<V>(x, static_cast<int>(at), c);
            W part = 0;
#pragma unroll
            for (int i = 0; i < V; ++i)
                part += static_cast<W>(v.v[i]);
            sum += part;
        }
        const W mean = static_cast<W>(row_total<kLongThreads>(sum, lds[0]) / c);
        for (int64_t at = t * V; at < c; at += kLongThreads * V)
        {
            const UVec<T, V> v = load<V>(x, static_cast<int>(at), c);
            W part = 0;
#pragma unroll
            for (int i = 0; i < V; ++i)
            {
                const W d = at + i < c ? static_cast<W>(v.v[i]) - mean : W(0);
                part = fma_(d, d, part);
            }
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
            const UVec<T, V> v = load<V>(x, static_cast<int>(at), c);
            using Alone = Shape<1, 1>; // (one vector at a time)
            UVec<P, V> w[1], b[1];
            load_weights<Alone, V>(a.scale ? a.scale + at : nullptr, 1.0f, 0, static_cast<int>(c - at), w);
            load_weights<Alone, V>(a.bias ? a.bias + at : nullptr, 0.0f, 0, static_cast<int>(c - at), b);
            W out[V];
#pragma unroll
            for (int i = 0; i < V; ++i)
                out[i] = fma_((static_cast<W>(v.v[i]) - mean) * rstd, static_cast<W>(w[0].v[i]), static_cast<W>(b[0].v[i]));
            store(y, static_cast<int>(at), c, out);
        }
        __syncthreads(); // (the sums' places are used again)
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
    uint32_t num_rows;
    int channels;
    bool streamed; // dx
};

// Rows in registers, as in the forward pass.  A thread keeps the sums for the gradients of its columns' weights; the sums of a workgroup's
// rows at a time meet in LDS at the end, in order.
template <typename T, typename P, typename S, bool Weights>
__global__ void __launch_bounds__(S::most_threads) ln_backward_kernel(const Backward<T, P> a)
{
    using W = wide<T>;
    constexpr int V = kVec<T>, K = S::vectors;
    constexpr bool kAhead = K * V <= 16;
    constexpr int kAtOnce = S::wave_rows ? kBlockSize / S::threads : 1; // rows
    __shared__ W lds[2][2][S::wave_rows ? 1 : S::threads / kWaveSize];
    const int t = threadIdx.x % S::threads, group = threadIdx.x / S::threads, c = a.channels;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * kAtOnce;
    uint64_t r = static_cast<uint64_t>(blockIdx.x) * kAtOnce + group;
    W dscale[Weights ? K : 1][V], dbias[Weights ? K : 1][V];
    if constexpr (Weights)
    {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
                dscale[k][i] = dbias[k][i] = W(0);
    }
    UVec<T, V> x[K], dy[K], next_x[kAhead ? K : 1], next_dy[kAhead ? K : 1];
    UVec<P, V> w[K];
    W mean = 0, rstd = 0, next_mean = 0, next_rstd = 0;
    const auto load_both = [&](uint32_t row, auto& to_x, auto& to_dy, W* to_mean, W* to_rstd) {
        load_row<S, V>(a.x + row_offset(a.x_rows, row), t, c, to_x);
        load_row<S, V>(a.dy + row_offset(a.dy_rows, row), t, c, to_dy);
        *to_mean = a.mean[row];
        *to_rstd = a.rstd[row];
    };
    load_weights<S, V>(a.scale, 1.0f, t, c, w);
    if (r < a.num_rows)
        load_both(static_cast<uint32_t>(r), x, dy, &mean, &rstd);
    // (all threads of a workgroup with one row at a time go round equally often)
    for (int turn = 0; r < a.num_rows; turn ^= 1)
    {
        const uint64_t following = r + step;
        const bool more = following < a.num_rows;
        if constexpr (kAhead)
        {
            if (more)
                load_both(static_cast<uint32_t>(following), next_x, next_dy, &next_mean, &next_rstd);
        }
        W h[K][V], g[K][V], sum = 0, dot = 0;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
            {
                // (behind the row's end dy is zero)
                h[k][i] = (static_cast<W>(x[k].v[i]) - mean) * rstd;
                g[k][i] = static_cast<W>(dy[k].v[i]);
                if constexpr (Weights)
                {
                    dscale[k][i] = fma_(g[k][i], h[k][i], dscale[k][i]);
                    dbias[k][i] += g[k][i];
                }
                g[k][i] *= static_cast<W>(w[k].v[i]);
                sum += g[k][i];
                dot = fma_(g[k][i], h[k][i], dot);
            }
        if (a.dx)
        {
            sum = row_total<S::threads>(sum, lds[turn][0]) / c;
            dot = row_total<S::threads>(dot, lds[turn][1]) / c;
            T* const dx = a.dx + row_offset(a.dx_rows, static_cast<uint32_t>(r));
#pragma unroll
            for (int k = 0; k < K; ++k)
            {
                const int at = (k * S::threads + t) * V;
                if (at >= c)
                    continue;
#pragma unroll
                for (int i = 0; i < V; ++i)
                    g[k][i] = rstd * (g[k][i] - fma_(h[k][i], dot, sum));
                store(dx, at, c, g[k], a.streamed);
            }
        }
        r = following;
        if constexpr (kAhead)
        {
#pragma unroll
            for (int k = 0; k < K; ++k)
            {
                x[k] = next_x[k];
                dy[k] = next_dy[k];
            }
            mean = next_mean;
            rstd = next_rstd;
        }
        else if (more)
            load_both(static_cast<uint32_t>(r), x, dy, &mean, &rstd);
    }
    if constexpr (Weights)
    {
        W* const out = a.partials + static_cast<size_t>(blockIdx.x) * c;
        const size_t half = static_cast<size_t>(gridDim.x) * c;
        if constexpr (S::wave_rows)
        {
            __shared__ W sums[kAtOnce - 1][S::threads * V];
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int which = 0; which < 2; ++which)
                {
                    W(&mine)[V] = which ? dbias[k] : dscale[k];
                    __syncthreads();
                    if (group > 0)
                    {
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            sums[group - 1][i * S::threads + t] = mine[i];
                    }
                    __syncthreads();
                    const int at = (k * S::threads + t) * V;
                    if (group == 0 && at < c)
                    {
#pragma unroll
                        for (int n = 0; n < kAtOnce - 1; ++n)
#pragma unroll
                            for (int i = 0; i < V; ++i)
                                mine[i] += sums[n][i * S::threads + t];
                        store(out + which * half, at, c, mine, a.streamed);
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
                    store(out, at, c, dscale[k], a.streamed);
                    store(out + half, at, c, dbias[k], a.streamed);
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
    for (uint32_t r = blockIdx.x; r < a.num_rows; r += gridDim.x)
    {
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
                const UVec<T, V> xs = load<V>(x, static_cast<int>(at), c), dys = load<V>(dy, static_cast<int>(at), c);
                UVec<P, V> w[1];
                load_weights<Shape<1, 1>, V>(a.scale ? a.scale + at : nullptr, 1.0f, 0, static_cast<int>(c - at), w);
                W out[V], s = 0, d = 0;
#pragma unroll
                for (int i = 0; i < V; ++i)
                {
                    const W h = (static_cast<W>(xs.v[i]) - mean) * rstd, g = static_cast<W>(dys.v[i]) * static_cast<W>(w[0].v[i]);
                    s += g;
                    d = fma_(g, h, d);
                    out[i] = rstd * (g - fma_(h, dot, sum));
                }
                sums += s;
                dots += d;
                if (pass == 1)
                    store(dx, static_cast<int>(at), c, out);
            }
            if (pass == 0)
            {
                sum = static_cast<W>(row_total<kLongThreads>(sums, lds[0]) / c);
                dot = static_cast<W>(row_total<kLongThreads>(dots, lds[1]) / c);
            }
        }
        __syncthreads(); // (the sums' places are used again)
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
        const UVec<T, V> x = load<V>(a.x + row_offset(a.x_rows, static_cast<uint32_t>(r)), at, c),
                         dy = load<V>(a.dy + row_offset(a.dy_rows, static_cast<uint32_t>(r)), at, c);
#pragma unroll
        for (int i = 0; i < V; ++i)
        {
            dscale[i] = fma_(static_cast<W>(dy.v[i]), (static_cast<W>(x.v[i]) - mean) * rstd, dscale[i]);
            dbias[i] += static_cast<W>(dy.v[i]);
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

constexpr int kMostChannels = 1 << 25; // (the weights' sums take 64 threads a channel, and a grid fewer than 2^32)

// How the rows are shared out: the fewest threads whose registers hold a row, one vector a thread below a wave, and 96 bytes of the sums' type a
// thread from there on, 64 in workgroups of 256 (the backward pass keeps four numbers an element, and the next row).  (Forward and backward
// in bf16, us, with a wave for rows of up to 2048 and 256 threads of up to 8192: 200000 x 32 62 and 169, 100000 x 300 37 and 104, 8192 x 2048
// 18 and 47, 4096 x 8192 26 and 83; so 11 and 26, 37 and 68, 17 and 34, 27 and 64.)
struct Split
{
    int threads, vectors; // of a row; threads = 0: too long for registers
};
constexpr int most_vectors(int vec, int threads)
{
    return threads < 64 ? 1 : (threads == 256 ? 64 : 96) / (vec == 2 ? 8 : 4) / vec;
}
Split split_rows(int vec, int channels)
{
    const int64_t vectors = (static_cast<int64_t>(channels) + vec - 1) / vec;
    for (const int threads : {8, 16, 32, 64, 256, 512})
    {
        const int64_t each = (vectors + threads - 1) / threads;
        if (each <= most_vectors(vec, threads))
            return {threads, static_cast<int>(each)};
    }
    return {0, 0};
}
constexpr int rows_at_once(int threads)
{
    return threads == 0 || threads > kWaveSize ? 1 : kBlockSize / threads;
}

// Outputs from 16 MiB on go past the caches, which keep the inputs: x is read by the backward pass again.  (Forward and backward of
// inputs that are not in the caches, with normal and with streaming stores: 4107 x 1155 floats, 18 MiB, 32.6 and 30.5 us; 32768 x 1024 in bf16, 64
// MiB, 95.8 and 95.9.)
bool is_streamed(size_t rows, int channels, size_t size)
{
    return rows * channels * size >= size_t(16) << 20;
}

// Workgroups whose sums for the weights' gradients are added up at the end: two for each CU where rows are that many, four where
// rows of a vector a thread leave registers for them.
uint32_t weight_parts(const Split& s, size_t num_rows)
{
    const size_t most = (s.threads > 0 && s.threads <= kWaveSize && s.vectors == 1 ? 4 : 2) * 256;
    const size_t groups = (num_rows + rows_at_once(s.threads) - 1) / rows_at_once(s.threads);
    return static_cast<uint32_t>(groups < most ? (groups ? groups : 1) : most);
}

// Workgroups for so many rows: as many as run at once, where rows are that many.
uint32_t workgroups(uint32_t rows, uint32_t rows_each, uint32_t threads)
{
    const uint32_t most = chip_units() * (2048 / threads), groups = static_cast<uint32_t>((static_cast<uint64_t>(rows) + rows_each - 1) / rows_each);
    return groups < most ? groups : most;
}

// f(Shape()) for rows of vectors of V elements.
template <int V, int Threads, int K, typename F>
int with_vectors(int vectors, const F& f)
{
    if constexpr (K < most_vectors(V, Threads))
    {
        if (vectors > K)
            return with_vectors<V, Threads, K + 1>(vectors, f);
    }
    return f(Shape<Threads, K>());
}
template <int V, typename F>
int with_shape(const Split& s, const F& f)
{
    return s.threads == 8     ? f(Shape<8, 1>())
           : s.threads == 16  ? f(Shape<16, 1>())
           : s.threads == 32  ? f(Shape<32, 1>())
           : s.threads == 64  ? with_vectors<V, 64, 1>(s.vectors, f)
           : s.threads == 256 ? with_vectors<V, 256, most_vectors(V, 64) / 4 + 1>(s.vectors, f)
                              : with_vectors<V, 512, most_vectors(V, 256) / 2 + 1>(s.vectors, f);
}

template <typename T, typename P>
int forward(const Forward<T, P>& a, hipStream_t stream)
{
    const Split s = split_rows(kVec<T>, a.channels);
    if (s.threads == 0)
    {
        launch(ln_forward_long_kernel<T, P>, dim3(workgroups(a.num_rows, 1, kLongThreads)), dim3(kLongThreads), stream, a);
        return launch_status();
    }
    return with_shape<kVec<T>>(s, [&](auto shape) {
        using S = decltype(shape);
        // a wave's rows: four waves a workgroup, one where rows are fewer than the waves that run at once
        const uint32_t waves = !S::wave_rows ? S::threads / kWaveSize : a.num_rows <= 4 * chip_units() ? 1 : kWavesPerBlock;
        const uint32_t rows = S::wave_rows ? waves * S::rows_of_wave : 1;
        launch(ln_forward_kernel<T, P, S>, dim3(workgroups(a.num_rows, rows, waves * kWaveSize)), dim3(waves * kWaveSize), stream, a);
        return launch_status();
    });
}

template <typename T, typename P>
int backward(const Backward<T, P>& a, P* dscale, P* dbias, hipStream_t stream)
{
    const Split s = split_rows(kVec<T>, a.channels);
    const bool weights = dscale || dbias;
    const uint32_t parts = weight_parts(s, a.num_rows);
    if (s.threads == 0)
    {
        if (weights) // first: dx may lie where x or dy does
        {
            const int64_t vectors = (static_cast<int64_t>(a.channels) + kVec<T> - 1) / kVec<T>;
            launch(ln_weights_long_kernel<T, P>, dim3(static_cast<uint32_t>((vectors + kBlockSize - 1) / kBlockSize), parts),
                   dim3(kBlockSize), stream, a);
        }
        if (a.dx && a.num_rows)
            launch(ln_backward_long_kernel<T, P>, dim3(workgroups(a.num_rows, 1, kLongThreads)), dim3(kLongThreads), stream, a);
    }
    else
    {
        (void) with_shape<kVec<T>>(s, [&](auto shape) {
            using S = decltype(shape);
            constexpr uint32_t kThreads = S::most_threads;
            if (weights)
                launch(ln_backward_kernel<T, P, S, true>, dim3(parts), dim3(kThreads), stream, a);
            else
                launch(ln_backward_kernel<T, P, S, false>, dim3(workgroups(a.num_rows, rows_at_once(S::threads), kThreads)),
                       dim3(kThreads), stream, a);
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
        if (num_rows > 0x7fffffffu || num_channels > kMostChannels)
            return H2X_ERR_TOO_LARGE;
        Forward<T, P> a{static_cast<const T*>(x), static_cast<const P*>(scale), static_cast<const P*>(bias),
                        static_cast<T*>(y),       static_cast<wide<T>*>(mean),  static_cast<wide<T>*>(rstd)};
        if (!make_rows(x_rows, num_rows, num_channels, &a.x_rows) || !make_rows(y_rows, num_rows, num_channels, &a.y_rows))
            return H2X_ERR_INVALID_ARGUMENT;
        if (num_rows == 0)
            return H2X_SUCCESS;
        if (!x || !y || (x == y && !alike(a.x_rows, a.y_rows)))
            return H2X_ERR_INVALID_ARGUMENT;
        a.num_rows = static_cast<uint32_t>(num_rows);
        a.channels = num_channels;
        a.epsilon = static_cast<wide<T>>(epsilon);
        a.streamed = is_streamed(num_rows, num_channels, sizeof(T));
        return forward(a, as_stream(stream));
    });
}

extern "C" size_t h2x_layer_norm_workspace_bytes(h2x_dtype dtype, size_t num_rows, int num_channels)
{
    const int size = element_size(dtype);
    if (size == 0 || num_channels < 1)
        return 0;
    const uint32_t parts = weight_parts(split_rows(16 / size, num_channels), num_rows);
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
        if (num_rows > 0x7fffffffu || num_channels > kMostChannels)
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
        if (dx && ((dx == x && !alike(a.dx_rows, a.x_rows)) || (dx == dy && !alike(a.dx_rows, a.dy_rows))))
            return H2X_ERR_INVALID_ARGUMENT;
        if (!weights && (!dx || num_rows == 0))
            return H2X_SUCCESS;
        a.num_rows = static_cast<uint32_t>(num_rows);
        a.channels = num_channels;
        a.streamed = is_streamed(num_rows, num_channels, sizeof(T));
        return backward(a, static_cast<P*>(dscale), static_cast<P*>(dbias), as_stream(stream));
    });
}
