// Attention, forward (include/h2x.h has the formulas; h2x_attention.hpp how the kernels are built).
//
// One pass over the keys with the running maximum and sum of each row's softmax, held by the row's lane.  The maximum is kept in
// units of log2 (scale * log2(e) times the score), so that a probability is one fused multiply-add and one exponential.
#include "h2x_attention.hpp"

namespace h2x
{
namespace attention
{
namespace
{

// Keys of a tile: 16 KB of 128 16-bit or 32-bit elements.
template <typename T>
constexpr int kTileKeys = sizeof(T) == 2 ? 64 : 32;

// What parts of the keys give, to be joined: for part p and row r (of samples * query_heads * queries), the unnormalised output at
// (p * rows + r) * padded_dim, and the row's maximum and sum at 2 (p * rows + r).
struct Parts
{
    float *out, *max_sum;
    int num; // 1: outputs are written at once
};

template <typename T>
struct Args
{
    const T *q, *k, *v;
    T* o;
    float* logsumexp; // or NULL
    Strides qs, ks, vs, os;
    Masks masks;
    Parts parts;
    float scale_log2;
    int dim, samples, query_heads, group, query_blocks;
    int heads; // of all samples; few queries: key heads
    Schedule schedule;
};

// A wave's 32 rows.
template <typename T, int DP>
struct Rows32
{
    Fragment<T, DP> q;
    f32x16 out[DP / 32]; // unnormalised
    float max, sum;      // the maximum in units of log2; the sum over this half's keys
    int from, end;       // keys that the lane's row sees

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
            out[d] = zero16();
        max = kLowest;
        sum = 0.0f;
    }

    // The scores of a tile's keys.
    __device__ __forceinline__ void score(LdsBytes k_tile, f32x16 (&s)[kTileKeys<T> / 32]) const
    {
        products<T, DP>(k_tile, 0, q, s);
    }

    // Scores to probabilities, with maximum, sum and output brought up to date.
    __device__ __forceinline__ void soften(f32x16 (&s)[kTileKeys<T> / 32], Weights<T> (&w)[kTileKeys<T> / 32], int first, bool masked,
                                           float scale_log2)
    {
        constexpr int B = kTileKeys<T> / 32;
        if (masked)
        {
#pragma unroll
            for (int b = 0; b < B; ++b)
                hide(&s[b], first + 32 * b, from, end);
        }
        float most = s[0][0];
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                most = fmaxf(most, s[b][i]);
        most = halves_max(most) * scale_log2;
        // The maximum that is subtracted may lie up to 2^8 below the true one: the sums have room for that, and the
        // output need not be rescaled at every tile.
        if (__any(most > max + 8.0f))
        {
            const float next = fmaxf(max, most), factor = __builtin_amdgcn_exp2f(max - next);
            max = next;
            sum *= factor;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    out[d][i] *= factor;
        }
        float part = 0.0f;
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], scale_log2, -max));
                part += p;
                w[b].set(i, p);
            }
        sum += part;
    }

    __device__ __forceinline__ void weigh(LdsBytes v_tile, const Weights<T> (&w)[kTileKeys<T> / 32])
    {
#pragma unroll
        for (int b = 0; b < kTileKeys<T> / 32; ++b)
            accumulate<DP>(v_tile, 32 * b, w[b], out);
    }
};

// Writes row `row` of the outputs (whose element 0 lies at o): what is there is out / sum, or a part's share.  max, sum: of the whole row.
template <typename T, int DP, bool Whole>
__device__ __forceinline__ void finish_row(const Args<T>& a, T* o, int64_t row, int part, const f32x16 (&out)[DP / 32],
                                           float max, float sum)
{
    const bool first_half = (threadIdx.x & 32) == 0;
    if (a.parts.num == 1)
    {
        store_row<T, DP, Whole>(o, a.dim, out, sum > 0.0f ? 1.0f / sum : 0.0f);
        if (a.logsumexp && first_half)
            a.logsumexp[row] = sum > 0.0f ? (max + log2f(sum)) * kLn2 : -INFINITY;
        return;
    }
    const int64_t rows = static_cast<int64_t>(a.samples) * a.query_heads * a.masks.queries, at = part * rows + row;
    if (first_half)
    {
        a.parts.max_sum[2 * at] = max;
        a.parts.max_sum[2 * at + 1] = sum;
    }
    if (sum > 0.0f)
        store_row<float, DP, true>(a.parts.out + at * DP, DP, out, 1.0f);
}

// Many queries: the waves of a workgroup take 32 queries of a head each, and share the tiles of keys and values, which come
// straight from memory to LDS while the tile before them is worked on.
template <typename T, int DP, bool Whole>
__global__ void __launch_bounds__(kThreads, 2) attention_forward_kernel(const Args<T> a)
{
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int KT = kTileKeys<T>, kTileBytes = KT * Tile<T, DP>::kRowBytes;
    __shared__ __attribute__((aligned(16))) char lds[2][2][kTileBytes];
    const Place place = place_of(a.schedule, blockIdx.x, gridDim.x, a.heads, a.query_blocks * a.parts.num);
    if (place.head >= a.heads)
        return;
    const int block = place.block / a.parts.num, part = place.block - block * a.parts.num;
    const int n = place.head / a.query_heads, head = place.head - n * a.query_heads;
    const int lane = threadIdx.x & (kWaveSize - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const Sample sample = sample_of(a.masks, n);

    // queries of the workgroup and of the wave
    const int block_first = block * (kWaves * kRows), block_end = min(block_first + kWaves * kRows, sample.queries);
    const int first = block_first + wave * kRows, i = first + (lane & 31);
    const int last = min(first + kRows, sample.queries) - 1; // (of the wave; before first: it has none)
    int from = 0, tiles = 0;
    if (block_first < block_end)
    {
        from = sample.first_key(block_first);
        tiles = (max(sample.end_key(block_end - 1) - from, 0) + KT - 1) / KT;
    }
    const int first_tile = static_cast<int>(static_cast<int64_t>(tiles) * part / a.parts.num);
    const int end_tile = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / a.parts.num);

    const T* const k = a.k + n * a.ks.sample + (head / a.group) * a.ks.head;
    const T* const v = a.v + n * a.vs.sample + (head / a.group) * a.vs.head;
    const int k_bytes = static_cast<int>(a.ks.token * sizeof(T)), v_bytes = static_cast<int>(a.vs.token * sizeof(T));
    const auto load = [&](int tile) {
        const int at = from + tile * KT, rows = min(KT, sample.keys - at);
        load_tile<T, DP, KT, kThreads, Whole>(buffer_of(k + at * a.ks.token, rows, a.ks.token, a.dim), k_bytes, a.dim,
                                              (LdsBytes) lds[tile & 1][0], threadIdx.x);
        load_tile<T, DP, KT, kThreads, Whole>(buffer_of(v + at * a.vs.token, rows, a.vs.token, a.dim), v_bytes, a.dim,
                                              (LdsBytes) lds[tile & 1][1], threadIdx.x);
    };
    if (first_tile < end_tile)
        load(first_tile);

    Rows32<T, DP> rows;
    rows.clear();
    load_fragment<T, DP, Whole>(&rows.q, a.q + n * a.qs.sample + head * a.qs.head + i * a.qs.token, i <= last, a.dim);
    rows.from = sample.first_key(min(i, max(last, 0)));
    rows.end = sample.end_key(min(i, max(last, 0)));
    // keys that some, and that all rows of the wave see
    const int some_from = sample.first_key(first), some_end = sample.end_key(last);
    const int all_from = sample.first_key(last), all_end = sample.end_key(first);

    for (int tile = first_tile; tile < end_tile; ++tile)
    {
        wait_for_loads();
        __syncthreads();
        if (tile + 1 < end_tile)
            load(tile + 1);
        const int at = from + tile * KT;
        if (first <= last && at < some_end && at + KT > some_from)
        {
            f32x16 s[KT / 32];
            Weights<T> w[KT / 32];
            rows.score((LdsBytes) lds[tile & 1][0], s);
            rows.soften(s, w, at, at < all_from || at + KT > all_end, a.scale_log2);
            rows.weigh((LdsBytes) lds[tile & 1][1], w);
        }
    }
    if (i < a.masks.queries)
    {
        const bool there = i < sample.queries;
        const float sum = halves_sum(rows.sum);
        finish_row<T, DP, Whole>(a, a.o + n * a.os.sample + head * a.os.head + i * a.os.token,
                                 (static_cast<int64_t>(n) * a.query_heads + head) * a.masks.queries + i, part, rows.out, rows.max,
                                 there ? sum : 0.0f);
    }
#endif
}

// Few queries: the queries of all heads that share a key head are rows of one wave's tile, so that keys and values are read once.
// The waves of a workgroup go through different tiles of the same part of the keys, each with LDS of its own and without barriers, and join what
// they have at the end.
template <typename T, int DP, bool Whole>
__global__ void __launch_bounds__(kThreads) attention_few_kernel(const Args<T> a)
{
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int KT = kTileKeys<T>, kTileBytes = KT * Tile<T, DP>::kRowBytes;
    constexpr int kLoads = KT * Tile<T, DP>::kChunks / kWaveSize; // of a wave, for a tile
    constexpr int kJoinStride = DP + 4;
    constexpr int kJoinBytes = kWaves * kRows * kJoinStride * 4, kTilesBytes = kWaves * 2 * kTileBytes;
    __shared__ __attribute__((aligned(16))) char lds[kTilesBytes > kJoinBytes ? kTilesBytes : kJoinBytes];
    __shared__ float max_sum[kWaves][kRows][2];
    const Place place = place_of({kByHead, 0}, blockIdx.x, gridDim.x, a.heads, a.query_blocks * a.parts.num);
    if (place.head >= a.heads)
        return;
    const int key_heads = a.query_heads / a.group;
    const int block = place.block / a.parts.num, part = place.block - block * a.parts.num;
    const int n = place.head / key_heads, key_head = place.head - n * key_heads;
    const int lane = threadIdx.x & (kWaveSize - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const Sample sample = sample_of(a.masks, n);

    // row r: query r % queries of the group's head r / queries
    const int queries = a.masks.queries, num_rows = a.group * queries;
    const int first = block * kRows, last = min(first + kRows, num_rows) - 1, r = min(first + (lane & 31), last);
    const int in_group = r / queries, i = r - in_group * queries, head = key_head * a.group + in_group;
    const bool one_head = first / queries == last / queries;
    const int first_query = one_head ? first - first / queries * queries : 0;
    const int last_query = min(one_head ? last - last / queries * queries : queries - 1, sample.queries - 1);
    int from = 0, tiles = 0;
    if (first_query <= last_query)
    {
        from = sample.first_key(first_query);
        tiles = (max(sample.end_key(last_query) - from, 0) + KT - 1) / KT;
    }
    const int first_tile = static_cast<int>(static_cast<int64_t>(tiles) * part / a.parts.num);
    const int end_tile = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / a.parts.num);

    const T* const k = a.k + n * a.ks.sample + key_head * a.ks.head;
    const T* const v = a.v + n * a.vs.sample + key_head * a.vs.head;
    const LdsBytes k_tile = (LdsBytes) (lds + wave * 2 * kTileBytes), v_tile = k_tile + kTileBytes;
    const auto load = [&](const T* p, const Strides& s, int tile, LdsBytes to) {
        const int at = from + tile * KT;
        load_tile<T, DP, KT, kWaveSize, Whole>(buffer_of(p + at * s.token, min(KT, sample.keys - at), s.token, a.dim),
                                               static_cast<int>(s.token * sizeof(T)), a.dim, to, lane);
    };

    Rows32<T, DP> rows;
    rows.clear();
    const bool there = i <= last_query;
    load_fragment<T, DP, Whole>(&rows.q, a.q + n * a.qs.sample + head * a.qs.head + i * a.qs.token, there, a.dim);
    rows.from = there ? sample.first_key(i) : 0;
    rows.end = there ? sample.end_key(i) : 0;
    const int all_from = sample.first_key(last_query), all_end = sample.end_key(first_query);

    int tile = first_tile + wave;
    if (tile < end_tile)
    {
        load(k, a.ks, tile, k_tile);
        load(v, a.vs, tile, v_tile);
    }
    for (; tile < end_tile; tile += kWaves)
    {
        const int at = from + tile * KT;
        f32x16 s[KT / 32];
        Weights<T> w[KT / 32];
        if constexpr (Whole)
            wait_for_loads<kLoads>(); // the keys are there, the values may be under way
        else
            wait_for_lds();
        rows.score(k_tile, s);
        wait_for_lds();
        const bool more = tile + kWaves < end_tile;
        if (more)
            load(k, a.ks, tile + kWaves, k_tile);
        // (a row beyond the sample's queries sees no key, and its wave no tile as a whole)
        rows.soften(s, w, at, at < all_from || at + KT > all_end, a.scale_log2);
        if constexpr (!Whole)
            wait_for_lds();
        else if (more)
            wait_for_loads<kLoads>();
        else
            wait_for_loads<0>();
        rows.weigh(v_tile, w);
        wait_for_lds();
        if (more)
            load(v, a.vs, tile + kWaves, v_tile);
    }

    // the waves' shares to LDS, and joined: thread t takes row t % 32 and every eighth run of four elements
    const float sum = halves_sum(rows.sum);
    if (lane < 32)
    {
        max_sum[wave][lane][0] = rows.max;
        max_sum[wave][lane][1] = sum;
    }
    __syncthreads(); // (no wave reads its tiles any more)
    float* const shares = reinterpret_cast<float*>(lds);
    store_row<float, DP, true>(shares + (wave * kRows + (lane & 31)) * kJoinStride, DP, rows.out, 1.0f);
    __syncthreads();
    const int row = threadIdx.x & 31, column = threadIdx.x / 32;
    float max = kLowest, total = 0.0f, factor[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
        max = fmaxf(max, max_sum[w][row][0]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
    {
        factor[w] = exp2f(max_sum[w][row][0] - max);
        total = __builtin_fmaf(max_sum[w][row][1], factor[w], total);
    }
    if (first + row > last)
        return;
    const int my_head = (first + row) / queries, my_query = first + row - my_head * queries;
    const bool mine = my_query < sample.queries;
    if (!mine)
        total = 0.0f;
    const int64_t at = (static_cast<int64_t>(n) * a.query_heads + key_head * a.group + my_head) * queries + my_query;
    const int64_t all = static_cast<int64_t>(a.samples) * a.query_heads * queries;
    const bool whole = a.parts.num == 1;
    T* const o = a.o + n * a.os.sample + (key_head * a.group + my_head) * a.os.head + my_query * a.os.token;
    float* const share = a.parts.out + (part * all + at) * DP;
    const float scale = total > 0.0f ? 1.0f / total : 0.0f;
    if (column == 0)
    {
        if (!whole)
        {
            a.parts.max_sum[2 * (part * all + at)] = max;
            a.parts.max_sum[2 * (part * all + at) + 1] = total;
        }
        else if (a.logsumexp)
            a.logsumexp[at] = total > 0.0f ? (max + log2f(total)) * kLn2 : -INFINITY;
    }
#pragma unroll
    for (int d = 4 * column; d < DP; d += 32)
    {
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
        {
            const f32x4 y = *reinterpret_cast<const f32x4*>(shares + (w * kRows + row) * kJoinStride + d);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[j] = __builtin_fmaf(y[j], factor[w], x[j]);
        }
        if (!whole)
        {
            *reinterpret_cast<f32x4*>(share + d) = x;
            continue;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (d + j < a.dim)
                o[d + j] = static_cast<T>(x[j] * scale);
    }
#endif
}

// Joins the parts of a row, a workgroup a row: a lane has a part's maximum and sum, a wave every fourth part's output.  (With a wave a row, one
// part after another, 512 rows of 16 parts took 21 us: a chain of waits for memory.)
constexpr int kMostParts = kWaveSize;
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) attention_join_kernel(const Args<T> a)
{
    constexpr int N = (DP + kWaveSize - 1) / kWaveSize; // elements of a lane
    __shared__ float outs[kWaves][N * kWaveSize], factors[kMostParts];
    const int64_t rows = static_cast<int64_t>(a.samples) * a.query_heads * a.masks.queries, row = blockIdx.x;
    const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
    float max = kLowest, sum = 0.0f;
    if (lane < a.parts.num)
    {
        max = a.parts.max_sum[2 * (lane * rows + row)];
        sum = a.parts.max_sum[2 * (lane * rows + row) + 1];
    }
    const bool any = sum > 0.0f; // (where no key was seen the output was not written)
    const float most = wave_combine(any ? max : kLowest, [](float x, float y) { return fmaxf(x, y); });
    const float factor = any ? __builtin_amdgcn_exp2f(max - most) : 0.0f;
    if (wave == 0)
        factors[lane] = factor;
    sum = token::wave_total(sum * factor);
    __syncthreads();
    float out[N] = {};
#pragma unroll 4
    for (int p = wave; p < a.parts.num; p += kWaves)
    {
        const float f = factors[p];
#pragma unroll
        for (int n = 0; n < N; ++n)
        {
            const float x = n * kWaveSize + lane < DP ? a.parts.out[(p * rows + row) * DP + n * kWaveSize + lane] : 0.0f;
            out[n] = f > 0.0f ? __builtin_fmaf(x, f, out[n]) : out[n];
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
        outs[wave][n * kWaveSize + lane] = out[n];
    __syncthreads();
    const int d = threadIdx.x;
    const int64_t of_head = row / a.masks.queries, i = row - of_head * a.masks.queries;
    const int64_t n = of_head / a.query_heads, head = of_head - n * a.query_heads;
    T* const o = a.o + n * a.os.sample + head * a.os.head + i * a.os.token;
    if (d < a.dim)
        o[d] = static_cast<T>(sum > 0.0f ? (outs[0][d] + outs[1][d] + outs[2][d] + outs[3][d]) / sum : 0.0f);
    if (a.logsumexp && d == 0)
        a.logsumexp[row] = sum > 0.0f ? (most + log2f(sum)) * kLn2 : -INFINITY;
}

// ---- host ------------------------------------------------------------------------------------------------------

// How a call is run.
struct Plan
{
    bool few;
    int query_blocks, parts, padded_dim;
    uint64_t groups; // workgroups
};

Plan plan_of(const h2x_attention& a)
{
    Plan p{};
    const int64_t group = a.query_heads / a.key_heads;
    p.few = a.queries <= 16;
    p.padded_dim = (a.head_dim + 31) / 32 * 32;
    const int64_t blocks = p.few ? (group * a.queries + kRows - 1) / kRows : (a.queries + kWaves * kRows - 1) / (kWaves * kRows);
    const int64_t groups = static_cast<int64_t>(a.samples) * (p.few ? a.key_heads : a.query_heads) * blocks;
    // The keys in parts while there are not workgroups for each CU several times, a part being eight tiles at least for each of
    // the waves that go through it one by one, or for the workgroup.
    const int tile = a.dtype == H2X_F32 ? 32 : 64;
    const int64_t least = p.few ? 4 * kWaves * tile : 8 * tile, aim = (p.few ? 8 : 2) * static_cast<int64_t>(chip_units());
    int64_t parts = 1;
    while (parts < kMostParts && groups * parts < aim && a.keys >= 2 * parts * least)
        parts *= 2;
    p.query_blocks = static_cast<int>(blocks);
    p.parts = static_cast<int>(parts);
    p.groups = static_cast<uint64_t>(groups) * parts;
    return p;
}

size_t rows_of(const h2x_attention& a)
{
    return static_cast<size_t>(a.samples) * a.query_heads * a.queries;
}

// Bytes of the parts' outputs, and of all.
size_t out_bytes(const h2x_attention& a, const Plan& p)
{
    return (p.parts * rows_of(a) * p.padded_dim * 4 + 255) & ~size_t(255);
}

template <typename T, bool Whole>
int issue(const h2x_attention& c, const Plan& p, const Args<T>& a, hipStream_t stream)
{
    const dim3 grid(static_cast<uint32_t>((p.groups + kNumXcd - 1) / kNumXcd * kNumXcd));
    return with_padded_dim(c.head_dim, [&](auto dim) {
        constexpr int DP = decltype(dim)::value;
        if (p.few)
            launch(attention_few_kernel<T, DP, Whole>, grid, dim3(kThreads), stream, a);
        else
            launch(attention_forward_kernel<T, DP, Whole>, grid, dim3(kThreads), stream, a);
        if (p.parts > 1)
            launch(attention_join_kernel<T, DP>, dim3(static_cast<uint32_t>(rows_of(c))), dim3(kThreads), stream, a);
        return launch_status();
    });
}

} // namespace
} // namespace attention
} // namespace h2x

using namespace h2x;
using namespace h2x::attention;

extern "C" size_t h2x_attention_forward_workspace_bytes(const h2x_attention* attention)
{
    if (check(attention) != H2X_SUCCESS || rows_of(*attention) == 0)
        return 0;
    const Plan p = plan_of(*attention);
    return p.parts == 1 ? 0 : out_bytes(*attention, p) + p.parts * rows_of(*attention) * 8;
}

extern "C" int h2x_attention_forward(const h2x_attention* attention, const void* q, const void* k, const void* v,
                                     const int32_t* query_lengths, const int32_t* key_lengths, void* o, float* logsumexp,
                                     void* workspace, h2x_stream_t stream)
{
    if (const int bad = check(attention))
        return bad;
    const h2x_attention& c = *attention;
    const Strides qs = strides_of(c, c.q, c.queries, c.query_heads), ks = strides_of(c, c.k, c.keys, c.key_heads),
                  vs = strides_of(c, c.v, c.keys, c.key_heads), os = strides_of(c, c.o, c.queries, c.query_heads);
    for (const int bad : {check_strides(c, qs, c.queries, c.query_heads, false), check_strides(c, ks, c.keys, c.key_heads, false),
                          check_strides(c, vs, c.keys, c.key_heads, false), check_strides(c, os, c.queries, c.query_heads, true)})
        if (bad)
            return bad;
    if (rows_of(c) == 0)
        return H2X_SUCCESS;
    const Plan p = plan_of(c);
    if (!q || !o || (c.keys > 0 && (!k || !v)) || (p.parts > 1 && !workspace))
        return H2X_ERR_INVALID_ARGUMENT;
    if (p.groups > 0x800000u || (p.parts > 1 && rows_of(c) > 0x800000u))
        return H2X_ERR_TOO_LARGE; // (a grid of fewer than 2^32 threads)
    const bool whole = whole_rows(c, q, qs) && whole_rows(c, k, ks) && whole_rows(c, v, vs) && whole_rows(c, o, os);
    return with_elements(c.dtype, whole, [&](auto t, auto is_whole) {
        using T = decltype(t);
        Args<T> a{};
        a.q = static_cast<const T*>(q);
        a.k = static_cast<const T*>(k);
        a.v = static_cast<const T*>(v);
        a.o = static_cast<T*>(o);
        a.logsumexp = logsumexp;
        a.qs = qs;
        a.ks = ks;
        a.vs = vs;
        a.os = os;
        a.masks = masks_of(c, query_lengths, key_lengths);
        a.parts.num = p.parts;
        a.parts.out = static_cast<float*>(workspace);
        if (p.parts > 1)
            a.parts.max_sum = reinterpret_cast<float*>(static_cast<char*>(workspace) + out_bytes(c, p));
        a.scale_log2 = static_cast<float>(c.scale * 1.4426950408889634);
        a.dim = c.head_dim;
        a.samples = c.samples;
        a.query_heads = c.query_heads;
        a.group = c.query_heads / c.key_heads;
        a.query_blocks = p.query_blocks;
        a.heads = c.samples * (p.few ? c.key_heads : c.query_heads);
        a.schedule = schedule_of(c, false, a.heads, static_cast<uint64_t>(p.query_blocks) * p.parts);
        return issue<T, decltype(is_whole)::value>(c, p, a, as_stream(stream));
    });
}
