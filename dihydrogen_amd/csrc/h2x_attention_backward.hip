// Attention, backward (include/h2x.h has the formulas; h2x_attention.hpp how the kernels are built).
//
// The probabilities are recomputed from the scores and the logarithms of the forward pass, in two passes: one over blocks of queries
// makes dq (and delta), one over blocks of keys dk and dv.  Each output is summed by the wave that writes it, in a fixed order; the
// price is that scores and d_o v^T are made twice, seven products in place of five.
#include "h2x_attention.hpp"

namespace h2x
{
namespace attention
{
namespace
{

// Rows of a tile that passes through LDS: 16 KB of 128 16-bit elements, 24 KB of floats.
template <typename T>
constexpr int kTileRows = sizeof(T) == 2 ? 64 : 32;

// Waves that a SIMD is to have: two, so that one's exponentials run beside the other's products, where 256 registers hold the rows.
template <typename T, int DP, bool Whole>
constexpr int kWavesOf = Whole && (sizeof(T) == 2 || DP <= 64) ? 2 : 1;

// With one wave a SIMD half of a lane's 512 registers are the matrix units' own: sums stay there from tile to tile.  (Left to itself the compiler
// moves all of them to and fro at each: 190 instructions of 700 for floats, heads of 96.)
template <int D>
__device__ __forceinline__ void keep_apart(f32x16 (&v)[D])
{
#ifdef __HIP_DEVICE_COMPILE__
#pragma unroll
    for (int d = 0; d < D; ++d)
        asm volatile("" : "+a"(v[d]));
#endif
}
template <int D>
__device__ __forceinline__ void keep_apart(f32x16 (&v)[D], f32x16 (&w)[D])
{
    keep_apart(v);
    keep_apart(w);
}

template <typename T>
struct Args
{
    const T *q, *k, *v, *o, *d_o;
    const float* logsumexp;
    T *dq, *dk, *dv;
    // of each row: its logarithm in units of log2 (the largest number where the row is empty), and delta
    float *log2_sum, *delta;
    Strides qs, ks, vs, os, d_os, dqs, dks, dvs;
    Masks masks;
    float scale, scale_log2;
    int dim, query_heads, group;
    int blocks, heads; // of rows in a head, and heads in all samples
    Order order;
    // The other side's tiles of a block of rows are shared by `parts` workgroups (1: one writes the gradients).  Part p's sums for row r, of `rows`, lie
    // at (p * rows + r) * padded_dim, those for the values behind those for the keys.
    int parts;
    float* partials;
};

// dq, and what the other pass needs of each row.  As in the forward pass, the waves of a workgroup take 32 queries of a head each.
template <typename T, int DP, int DQ, bool Whole>
__global__ void __launch_bounds__(kThreads, (kWavesOf<T, DP, Whole>)) attention_dq_kernel(const Args<T> a)
{
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int KT = kTileRows<T>, B = KT / 32;
    __shared__ __attribute__((aligned(16))) char lds[2][2][kTileBytes<T, DP, KT>];
    const Place place = place_of(a.order, blockIdx.x, gridDim.x, a.heads, a.blocks * a.parts);
    if (place.head >= a.heads)
        return;
    const int block = place.block / a.parts, part = place.block - block * a.parts;
    const int n = place.head / a.query_heads, head = place.head - n * a.query_heads;
    const int lane = threadIdx.x & (kWaveSize - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const Sample sample = sample_of(a.masks, n);

    const int block_first = block * (kWaves * kRows), block_end = min(block_first + kWaves * kRows, sample.queries);
    const int first = block_first + wave * kRows, i = first + (lane & 31);
    const int last = min(first + kRows, sample.queries) - 1;
    // keys that some row of the workgroup sees; what else lies in their tiles is read as zero
    int from = 0, to = 0;
    if (block_first < block_end)
    {
        from = sample.first_key(block_first);
        to = sample.end_key(block_end - 1);
    }
    const int tiles = (max(to - from, 0) + KT - 1) / KT;
    const int first_tile = static_cast<int>(static_cast<int64_t>(tiles) * part / a.parts);
    const int end_tile = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / a.parts);
    const T* const k = a.k + n * a.ks.sample + (head / a.group) * a.ks.head;
    const T* const v = a.v + n * a.vs.sample + (head / a.group) * a.vs.head;
    const int k_bytes = static_cast<int>(a.ks.token * sizeof(T)), v_bytes = static_cast<int>(a.vs.token * sizeof(T));
    TileLoad<T, DP, KT, kThreads, Whole> k_load, v_load;
    const auto issue = [&](int tile) {
        const int at = from + tile * KT, rows = min(KT, to - at);
        k_load.issue(buffer_of(k + at * a.ks.token, rows, a.ks.token, a.dim), k_bytes, a.dim, (LdsBytes) lds[tile & 1][0],
                     threadIdx.x);
        v_load.issue(buffer_of(v + at * a.vs.token, rows, a.vs.token, a.dim), v_bytes, a.dim, (LdsBytes) lds[tile & 1][1],
                     threadIdx.x);
    };
    const auto put = [&](int tile) {
        k_load.put((LdsBytes) lds[tile & 1][0], threadIdx.x);
        v_load.put((LdsBytes) lds[tile & 1][1], threadIdx.x);
    };
    if (first_tile < end_tile)
    {
        issue(first_tile);
        put(first_tile);
    }

    const int row_from = sample.first_key(min(i, max(last, 0))), row_end = sample.end_key(min(i, max(last, 0)));
    const bool there = i <= last && row_from < row_end; // (a row that sees no key may hold anything)
    const int64_t row = (static_cast<int64_t>(n) * a.query_heads + head) * a.masks.queries + i;
    Fragment<T, DQ> q, d_o;
    float delta = 0.0f, log2_sum = -kLowest;
    {
        const T* const o_row = a.o + n * a.os.sample + head * a.os.head + i * a.os.token;
        const T* const d_o_row = a.d_o + n * a.d_os.sample + head * a.d_os.head + i * a.d_os.token;
#pragma unroll
        for (int c = 0; c < DQ / 16; ++c)
        {
            const int at = 16 * c + 8 * (lane / 32);
            const Eight<T> x = load_eight<T, Whole>(o_row, at, there, a.dim), y = load_eight<T, Whole>(d_o_row, at, there, a.dim);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                delta = __builtin_fmaf(element(x, e), element(y, e), delta);
            planes_of(y, d_o.chunk[c]);
        }
        delta = halves_sum(delta);
    }
    load_fragment<T, DQ, Whole>(&q, a.q + n * a.qs.sample + head * a.qs.head + i * a.qs.token, there, a.dim);
    if (there)
    {
        const float l = a.logsumexp[row];
        if (l != -INFINITY) // (one that is NaN is no empty row's)
            log2_sum = l * kLog2e;
        if (lane < 32 && part == 0)
        {
            a.log2_sum[row] = log2_sum;
            a.delta[row] = delta;
        }
    }
    f32x16 dq[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
        dq[d] = zero16();
    const int some_from = sample.first_key(first), some_end = sample.end_key(last);
    const int all_from = sample.first_key(last), all_end = sample.end_key(first);

    for (int tile = first_tile; tile < end_tile; ++tile)
    {
        wait_for_loads();
        __syncthreads();
        if (tile + 1 < end_tile)
            issue(tile + 1);
        const LdsBytes k_tile = (LdsBytes) lds[tile & 1][0], v_tile = (LdsBytes) lds[tile & 1][1];
        const int at = from + tile * KT;
        if (first <= last && at < some_end && at + KT > some_from)
        {
            f32x16 s[B], dp[B];
            products<T, DP, DQ, KT>(k_tile, 0, q, s);
            products<T, DP, DQ, KT>(v_tile, 0, d_o, dp);
            if (at < all_from || at + KT > all_end)
            {
#pragma unroll
                for (int b = 0; b < B; ++b)
                    hide(&s[b], at + 32 * b, row_from, row_end);
            }
            Weights<T> ds[B];
#pragma unroll
            for (int b = 0; b < B; ++b)
            {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    s[b][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][j], a.scale_log2, -log2_sum)) * (dp[b][j] - delta);
#pragma unroll
                for (int j = 0; j < 16; j += 2)
                    ds[b].set(j, s[b][j], s[b][j + 1]);
            }
#pragma unroll
            for (int b = 0; b < B; ++b)
                accumulate<T, DP, KT>(k_tile, 32 * b, ds[b], dq);
        }
        if (tile + 1 < end_tile)
            put(tile + 1); // (all waves are past the tile that lay there)
        if constexpr (kWavesOf<T, DP, Whole> == 1)
            keep_apart(dq);
    }
    if (i >= a.masks.queries)
        return;
    if (a.parts > 1)
        store_row<float, DP, true>(
            a.partials + (static_cast<int64_t>(part) * a.heads * a.masks.queries + row) * DP, DP, dq, 1.0f);
    else
        store_row<T, DP, Whole>(a.dq + n * a.dqs.sample + head * a.dqs.head + i * a.dqs.token, a.dim, dq, a.scale);
#endif
}

// dk and dv: the waves of a workgroup take 32 keys of a key head each; the queries of the heads that share it pass through LDS, one head after
// another.
template <typename T, int DP, int DQ, bool Whole>
__global__ void __launch_bounds__(kThreads, (DP == 128 ? 1 : kWavesOf<T, DP, Whole>)) attention_dkv_kernel(const Args<T> a)
{
#ifdef __HIP_DEVICE_COMPILE__
    constexpr bool kOneWave = DP == 128 || kWavesOf<T, DP, Whole> == 1; // (128 elements: two waves would have to spill)
    constexpr int QT = kTileRows<T>, B = QT / 32, N = DP <= 64 ? 1 : B; // blocks at a time
    __shared__ __attribute__((aligned(16))) char lds[2][2][kTileBytes<T, DP, QT>];
    __shared__ __attribute__((aligned(16))) float stats[2][2][kWaveSize];
    const int key_heads = a.query_heads / a.group;
    const Place place = place_of(a.order, blockIdx.x, gridDim.x, a.heads, a.blocks * a.parts);
    if (place.head >= a.heads)
        return;
    const int block = place.block / a.parts, part = place.block - block * a.parts;
    const int n = place.head / key_heads, key_head = place.head - n * key_heads;
    const int lane = threadIdx.x & (kWaveSize - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const Sample sample = sample_of(a.masks, n);

    const int block_first = block * (kWaves * kRows), block_end = min(block_first + kWaves * kRows, sample.keys);
    const int first = block_first + wave * kRows, j = first + (lane & 31);
    const int last = min(first + kRows, sample.keys) - 1;
    int from = 0, to = 0;
    if (block_first < block_end)
    {
        from = sample.first_query(block_first);
        to = sample.end_query(block_end - 1);
    }
    const int tiles = (max(to - from, 0) + QT - 1) / QT;
    const int q_bytes = static_cast<int>(a.qs.token * sizeof(T)), d_o_bytes = static_cast<int>(a.d_os.token * sizeof(T));
    TileLoad<T, DP, QT, kThreads, Whole> q_load, d_o_load;
    // tile `tile` of the group's head `g`, to stage `stage`
    const auto issue = [&](int g, int tile, int stage) {
        const int head = key_head * a.group + g, at = from + tile * QT, rows = min(QT, to - at);
        const T* const q = a.q + n * a.qs.sample + head * a.qs.head + at * a.qs.token;
        const T* const d_o = a.d_o + n * a.d_os.sample + head * a.d_os.head + at * a.d_os.token;
        q_load.issue(buffer_of(q, rows, a.qs.token, a.dim), q_bytes, a.dim, (LdsBytes) lds[stage][0], threadIdx.x);
        d_o_load.issue(buffer_of(d_o, rows, a.d_os.token, a.dim), d_o_bytes, a.dim, (LdsBytes) lds[stage][1], threadIdx.x);
        // rows' logarithms by one wave, their deltas by another (zero behind the sample's queries, as q and d_o are)
        if (wave < 2)
        {
            const float* const p = (wave == 0 ? a.log2_sum : a.delta)
                                   + (static_cast<int64_t>(n) * a.query_heads + head) * a.masks.queries + at;
            load_to_lds<4>(buffer_of(p, rows, 1, 1), 4 * lane, (LdsBytes) stats[stage][wave]);
        }
    };
    const auto put = [&](int stage) {
        q_load.put((LdsBytes) lds[stage][0], threadIdx.x);
        d_o_load.put((LdsBytes) lds[stage][1], threadIdx.x);
    };
    const int64_t all_steps = static_cast<int64_t>(tiles) * a.group;
    const int first_step = static_cast<int>(all_steps * part / a.parts), steps = static_cast<int>(all_steps * (part + 1) / a.parts);
    int g = tiles > 0 ? first_step / tiles : 0, tile = first_step - g * tiles;
    if (first_step < steps)
    {
        issue(g, tile, first_step & 1);
        put(first_step & 1);
    }

    const int row_from = sample.first_query(min(j, max(last, 0))), row_end = sample.end_query(min(j, max(last, 0)));
    const bool there = j <= last && row_from < row_end; // (a key that no query sees may hold anything)
    Fragment<T, DQ> k, v;
    load_fragment<T, DQ, Whole>(&k, a.k + n * a.ks.sample + key_head * a.ks.head + j * a.ks.token, there, a.dim);
    load_fragment<T, DQ, Whole>(&v, a.v + n * a.vs.sample + key_head * a.vs.head + j * a.vs.token, there, a.dim);
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
        dk[d] = dv[d] = zero16();
    const int some_from = sample.first_query(first), some_end = sample.end_query(last);
    const int all_from = sample.first_query(last), all_end = sample.end_query(first);

    for (int step = first_step; step < steps; ++step)
    {
        const int stage = step & 1, here = from + tile * QT;
        wait_for_loads();
        __syncthreads();
        if (++tile == tiles)
            tile = 0, ++g;
        if (step + 1 < steps)
            issue(g, tile, stage ^ 1);
        const LdsBytes q_tile = (LdsBytes) lds[stage][0], d_o_tile = (LdsBytes) lds[stage][1];
        const float* const log2_sum = &stats[stage][0][4 * (lane / 32)];
        const float* const delta = &stats[stage][1][4 * (lane / 32)];
#pragma unroll
        for (int b0 = 0; b0 < B; b0 += N)
        {
            const int at = here + 32 * b0;
            if (first > last || at >= some_end || at + 32 * N <= some_from)
                continue;
            // (Where two blocks are taken in one go, the products of one run beside the exponentials of the other.)
            f32x16 s[N], dp[N];
            products<T, DP, DQ, QT>(q_tile, 32 * b0, k, s);
            products<T, DP, DQ, QT>(d_o_tile, 32 * b0, v, dp);
            if (at < all_from || at + 32 * N > all_end)
            {
#pragma unroll
                for (int b = 0; b < N; ++b)
                    hide(&s[b], at + 32 * b, row_from, row_end);
            }
            Weights<T> p[N], ds[N];
#pragma unroll
            for (int b = 0; b < N; ++b)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                {
                    const f32x4 l = *reinterpret_cast<const f32x4*>(log2_sum + 32 * (b0 + b) + 2 * r);
                    const f32x4 m = *reinterpret_cast<const f32x4*>(delta + 32 * (b0 + b) + 2 * r);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                    {
                        s[b][r + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r + e], a.scale_log2, -l[e]));
                        dp[b][r + e] = s[b][r + e] * (dp[b][r + e] - m[e]);
                    }
                    p[b].set(r, s[b][r], s[b][r + 1]);
                    p[b].set(r + 2, s[b][r + 2], s[b][r + 3]);
                    ds[b].set(r, dp[b][r], dp[b][r + 1]);
                    ds[b].set(r + 2, dp[b][r + 2], dp[b][r + 3]);
                }
#pragma unroll
            for (int b = 0; b < N; ++b)
            {
                accumulate<T, DP, QT>(d_o_tile, 32 * (b0 + b), p[b], dv);
                accumulate<T, DP, QT>(q_tile, 32 * (b0 + b), ds[b], dk);
            }
        }
        if (step + 1 < steps)
            put(stage ^ 1);
        if constexpr (kOneWave)
            keep_apart(dk, dv);
    }
    if (j < a.masks.keys)
    {
        if (!there) // (a key of zeros may have had infinite weights)
        {
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
                dk[d] = dv[d] = zero16();
        }
        if (a.parts > 1)
        {
            const int64_t rows = static_cast<int64_t>(a.heads) * a.masks.keys;
            float* const p = a.partials + (part * rows + static_cast<int64_t>(place.head) * a.masks.keys + j) * DP;
            store_row<float, DP, true>(p, DP, dk, 1.0f);
            store_row<float, DP, true>(p + a.parts * rows * DP, DP, dv, 1.0f);
            return;
        }
        store_row<T, DP, Whole>(a.dk + n * a.dks.sample + key_head * a.dks.head + j * a.dks.token, a.dim, dk, a.scale);
        store_row<T, DP, Whole>(a.dv + n * a.dvs.sample + key_head * a.dvs.head + j * a.dvs.token, a.dim, dv, 1.0f);
    }
#endif
}

// Sums of the parts of gradients, in the parts' order: four elements of a row a thread.
template <typename T>
struct Sum
{
    const float* partials;
    T* out[2]; // of grid.y
    Strides strides[2];
    float factor[2];
    int parts, padded_dim, dim, tokens, heads; // heads of a sample
    int64_t rows;
};
template <typename T>
__global__ void __launch_bounds__(kThreads) attention_sum_kernel(const Sum<T> a)
{
    const int fours = a.padded_dim / 4, which = blockIdx.y;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, row = at / fours;
    const int d = static_cast<int>(at - row * fours) * 4;
    if (row >= a.rows || d >= a.dim)
        return;
    const float* p = a.partials + (which * static_cast<int64_t>(a.parts) * a.rows + row) * a.padded_dim + d;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int part = 0; part < a.parts; ++part, p += a.rows * a.padded_dim)
        sum += *reinterpret_cast<const f32x4*>(p);
    const int64_t of_head = row / a.tokens, i = row - of_head * a.tokens, n = of_head / a.heads, head = of_head - n * a.heads;
    T* const out = a.out[which] + n * a.strides[which].sample + head * a.strides[which].head + i * a.strides[which].token + d;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (d + e < a.dim)
            out[e] = static_cast<T>(sum[e] * a.factor[which]);
}

// ---- host ------------------------------------------------------------------------------------------------------

size_t rows_of(const h2x_attention& a)
{
    return static_cast<size_t>(a.samples) * a.query_heads * a.queries;
}

// How a call is run.
struct Plan
{
    uint64_t query_blocks, key_blocks; // of a head
    int query_parts, key_parts;
    size_t partials_bytes, bytes; // of the workspace: of the partial sums, and of all
};

// The other side's tiles in parts, while workgroups are fewer than CUs (twice as many under a mask that bounds one side, where they are of unlike
// lengths), 16 tiles a part at least.  (Without and with parts, bf16: 8 query heads over one key head, 4096 tokens of 128, causal,
// 1082 and 196 us; 16384 queries and 77 keys, 8 heads of 64, 370 and 57; 100 queries and 16384 keys, 2 heads, 276 and 36.)
int parts_of(const h2x_attention& a, uint64_t groups, uint64_t tiles)
{
    const uint64_t most = ((a.window_left < 0) != (a.window_right < 0) ? 2 : 1) * static_cast<uint64_t>(chip_units());
    int parts = 1;
    while (parts < 64 && groups * parts * 2 <= most && tiles >= 32u * parts)
        parts *= 2;
    return parts;
}

Plan plan_of(const h2x_attention& a)
{
    const uint64_t rows = kWaves * kRows, tile = a.dtype == H2X_F32 ? 32 : 64;
    Plan p{};
    p.query_blocks = (a.queries + rows - 1) / rows;
    p.key_blocks = (a.keys + rows - 1) / rows;
    p.query_parts = parts_of(a, p.query_blocks * a.samples * a.query_heads, (a.keys + tile - 1) / tile);
    p.key_parts = parts_of(a, p.key_blocks * a.samples * a.key_heads, (a.queries + tile - 1) / tile * (a.query_heads / a.key_heads));
    const size_t dim = (a.head_dim + 31) / 32 * 32 * 4;
    const size_t of_queries = p.query_parts > 1 ? p.query_parts * rows_of(a) * dim : 0;
    const size_t of_keys = p.key_parts > 1 ? 2 * p.key_parts * static_cast<size_t>(a.samples) * a.key_heads * a.keys * dim : 0;
    p.partials_bytes = of_queries > of_keys ? of_queries : of_keys; // (one after the other)
    p.bytes = p.partials_bytes + 8 * rows_of(a);
    return p;
}

template <typename T, bool Whole>
int issue(const h2x_attention& c, const Plan& p, Args<T> a, hipStream_t stream)
{
    const uint64_t query_heads = static_cast<uint64_t>(c.samples) * c.query_heads, key_heads = static_cast<uint64_t>(c.samples) * c.key_heads;
    const uint64_t query_groups = p.query_blocks * p.query_parts * query_heads, key_groups = p.key_blocks * p.key_parts * key_heads;
    if (query_groups > 0x800000u || key_groups > 0x800000u) // a grid of fewer than 2^32 threads
        return H2X_ERR_TOO_LARGE;
    const auto grid = [](uint64_t groups) { return dim3(static_cast<uint32_t>((groups + kNumXcd - 1) / kNumXcd * kNumXcd)); };
    return with_padded_dim(c.head_dim, [&](auto dim) {
        constexpr int DP = decltype(dim)::in_lds, DQ = decltype(dim)::contracted;
        Sum<T> sum{a.partials, {}, {}, {a.scale, 1.0f}, 0, DP, c.head_dim, 0, 0, 0};
        const auto join = [&](int outputs) {
            launch(attention_sum_kernel<T>, dim3(static_cast<uint32_t>((sum.rows * (DP / 4) + kThreads - 1) / kThreads), outputs),
                   dim3(kThreads), stream, sum);
        };
        if (query_groups > 0)
        {
            a.blocks = static_cast<int>(p.query_blocks);
            a.heads = static_cast<int>(query_heads);
            a.parts = p.query_parts;
            a.order = order_of(c, false);
            launch(attention_dq_kernel<T, DP, DQ, Whole>, grid(query_groups), dim3(kThreads), stream, a);
            if (a.parts > 1)
            {
                sum.out[0] = a.dq;
                sum.strides[0] = a.dqs;
                sum.parts = a.parts;
                sum.tokens = static_cast<int>(c.queries);
                sum.heads = c.query_heads;
                sum.rows = static_cast<int64_t>(rows_of(c));
                join(1);
            }
        }
        if (key_groups > 0)
        {
            a.blocks = static_cast<int>(p.key_blocks);
            a.heads = static_cast<int>(key_heads);
            a.parts = p.key_parts;
            a.order = order_of(c, true);
            launch(attention_dkv_kernel<T, DP, DQ, Whole>, grid(key_groups), dim3(kThreads), stream, a);
            if (a.parts > 1)
            {
                sum.out[0] = a.dk;
                sum.out[1] = a.dv;
                sum.strides[0] = a.dks;
                sum.strides[1] = a.dvs;
                sum.parts = a.parts;
                sum.tokens = static_cast<int>(c.keys);
                sum.heads = c.key_heads;
                sum.rows = static_cast<int64_t>(key_heads) * c.keys;
                join(2);
            }
        }
        return launch_status();
    });
}

} // namespace
} // namespace attention
} // namespace h2x

using namespace h2x;
using namespace h2x::attention;

extern "C" size_t h2x_attention_backward_workspace_bytes(const h2x_attention* attention)
{
    if (check(attention) != H2X_SUCCESS || attention->samples == 0 || attention->query_heads == 0)
        return 0; // (without query heads: zeros alone are written)
    return plan_of(*attention).bytes;
}

extern "C" int h2x_attention_backward(const h2x_attention* attention, const void* q, const void* k, const void* v, const void* o,
                                      const void* d_o, const float* logsumexp, const int32_t* query_lengths,
                                      const int32_t* key_lengths, void* dq, void* dk, void* dv, void* workspace,
                                      h2x_stream_t stream)
{
    if (const int bad = check(attention))
        return bad;
    h2x_attention c = *attention;
    struct Operand
    {
        const void* p;
        const h2x_token_strides* given;
        int64_t tokens;
        int heads;
        bool output;
        Strides s;
    } operands[] = {{q, &c.q, c.queries, c.query_heads, false},     {k, &c.k, c.keys, c.key_heads, false},
                    {v, &c.v, c.keys, c.key_heads, false},          {o, &c.o, c.queries, c.query_heads, false},
                    {d_o, &c.d_o, c.queries, c.query_heads, false}, {dq, &c.dq, c.queries, c.query_heads, true},
                    {dk, &c.dk, c.keys, c.key_heads, true},         {dv, &c.dv, c.keys, c.key_heads, true}};
    bool whole = true, missing = false;
    for (Operand& x : operands)
    {
        x.s = strides_of(c, *x.given, x.tokens, x.heads);
        if (const int bad = check_strides(c, x.s, x.tokens, x.heads, x.output))
            return bad;
        whole = whole && whole_rows(c, x.p, x.s);
        missing = missing || (!x.p && x.tokens > 0 && x.heads > 0);
    }
    if (c.query_heads == 0) // keys have the gradients that they have from no queries
    {
        c.query_heads = c.key_heads;
        c.queries = 0;
    }
    if (c.samples == 0 || c.key_heads == 0 || (c.queries == 0 && c.keys == 0))
        return H2X_SUCCESS;
    for (int out = 5; out < 8; ++out) // the second kernel reads what the first would have overwritten
        for (int x = 0; x < out; ++x)
            if (operands[out].p && operands[out].p == operands[x].p)
                return H2X_ERR_INVALID_ARGUMENT;
    const Plan p = plan_of(c);
    if (missing || (c.queries > 0 && !logsumexp) || (p.bytes > 0 && !workspace))
        return H2X_ERR_INVALID_ARGUMENT;
    if ((c.queries + 31) / 32 * (c.query_heads / c.key_heads) > 0x7fffffff)
        return H2X_ERR_TOO_LARGE;
    return with_elements(c.dtype, whole, [&](auto t, auto is_whole) {
        using T = decltype(t);
        Args<T> a{};
        a.q = static_cast<const T*>(q);
        a.k = static_cast<const T*>(k);
        a.v = static_cast<const T*>(v);
        a.o = static_cast<const T*>(o);
        a.d_o = static_cast<const T*>(d_o);
        a.logsumexp = logsumexp;
        a.dq = static_cast<T*>(dq);
        a.dk = static_cast<T*>(dk);
        a.dv = static_cast<T*>(dv);
        a.partials = static_cast<float*>(workspace);
        a.log2_sum = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.partials_bytes);
        a.delta = a.log2_sum + rows_of(c);
        Strides* const strides[] = {&a.qs, &a.ks, &a.vs, &a.os, &a.d_os, &a.dqs, &a.dks, &a.dvs};
        for (int i = 0; i < 8; ++i)
            *strides[i] = operands[i].s;
        a.masks = masks_of(c, query_lengths, key_lengths);
        a.scale = static_cast<float>(c.scale);
        a.scale_log2 = static_cast<float>(c.scale * 1.4426950408889634);
        a.dim = c.head_dim;
        a.query_heads = c.query_heads;
        a.group = c.query_heads / c.key_heads;
        return issue<T, decltype(is_whole)::value>(c, p, a, as_stream(stream));
    });
}
