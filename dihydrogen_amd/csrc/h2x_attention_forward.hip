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

// Keys of a tile: 16 KB of 128 16-bit elements, 24 KB of floats.
template <typename T>
constexpr int kTileKeys = sizeof(T) == 2 ? 64 : 32;

// What parts of the keys give, to be joined: for part p and row r (of samples * query_heads * queries), the unnormalised output at
// (p * rows + r) * padded_dim, and the row's maximum and sum at 2 (p * rows + r).  The maximum of a row that sees no key of any part is minus
// infinity; of one that sees some it is finite in parts where it sees none.
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
    int heads; // of all samples; with split keys key heads
    Order order;
};

// A wave's 32 rows.
template <typename T, int DP, int DQ>
struct Rows32
{
    Fragment<T, DQ> q;
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
        products<T, DP, DQ, kTileKeys<T>>(k_tile, 0, q, s);
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
            for (int i = 0; i < 16; i += 2)
            {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], scale_log2, -max));
                const float q = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i + 1], scale_log2, -max));
                part += p;
                part += q;
                w[b].set(i, p, q);
            }
        sum += part;
    }

    __device__ __forceinline__ void weigh(LdsBytes v_tile, const Weights<T> (&w)[kTileKeys<T> / 32])
    {
#pragma unroll
        for (int b = 0; b < kTileKeys<T> / 32; ++b)
            accumulate<T, DP, kTileKeys<T>>(v_tile, 32 * b, w[b], out);
    }
};

// Many queries: the waves of a workgroup take 32 queries of a head each, and share the tiles of keys and values, which come
// straight from memory to LDS while the tile before them is worked on.
template <typename T, int DP, int DQ, bool Whole>
__global__ void __launch_bounds__(kThreads, (sizeof(T) == 2 || DP <= 96 ? 2 : 1)) attention_forward_kernel(const Args<T> a)
{
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int KT = kTileKeys<T>;
    __shared__ __attribute__((aligned(16))) char lds[2][2][kTileBytes<T, DP, KT>];
    const Place place = place_of(a.order, blockIdx.x, gridDim.x, a.heads, a.query_blocks);
    if (place.head >= a.heads)
        return;
    const int block = place.block, n = place.head / a.query_heads, head = place.head - n * a.query_heads;
    const int lane = threadIdx.x & (kWaveSize - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const Sample sample = sample_of(a.masks, n);

    // queries of the workgroup and of the wave
    const int block_first = block * (kWaves * kRows), block_end = min(block_first + kWaves * kRows, sample.queries);
    const int first = block_first + wave * kRows, i = first + (lane & 31);
    const int last = min(first + kRows, sample.queries) - 1; // (of the wave; before first: it has none)
    // keys that some row of the workgroup sees; what else lies in their tiles is read as zero
    int from = 0, to = 0;
    if (block_first < block_end)
    {
        from = sample.first_key(block_first);
        to = sample.end_key(block_end - 1);
    }
    const int tiles = (max(to - from, 0) + KT - 1) / KT;
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
    if (tiles > 0)
    {
        issue(0);
        put(0);
    }

    Rows32<T, DP, DQ> rows;
    rows.clear();
    load_fragment<T, DQ, Whole>(&rows.q, a.q + n * a.qs.sample + head * a.qs.head + i * a.qs.token, i <= last, a.dim);
    rows.from = sample.first_key(min(i, max(last, 0)));
    rows.end = sample.end_key(min(i, max(last, 0)));
    // keys that some, and that all rows of the wave see
    const int some_from = sample.first_key(first), some_end = sample.end_key(last);
    const int all_from = sample.first_key(last), all_end = sample.end_key(first);

    for (int tile = 0; tile < tiles; ++tile)
    {
        wait_for_loads();
        __syncthreads();
        if (tile + 1 < tiles)
            issue(tile + 1);
        const int at = from + tile * KT;
        if (first <= last && at < some_end && at + KT > some_from)
        {
            f32x16 s[KT / 32];
            Weights<T> w[KT / 32];
            rows.score((LdsBytes) lds[tile & 1][0], s);
            rows.soften(s, w, at, at < all_from || at + KT > all_end, a.scale_log2);
            rows.weigh((LdsBytes) lds[tile & 1][1], w);
        }
        if (tile + 1 < tiles)
            put(tile + 1); // (all waves are past the tile that lay there)
    }
    if (i < a.masks.queries)
    {
        const bool sees = i < sample.queries && rows.from < rows.end; // (its sum may still be anything, NaN among them)
        const float sum = halves_sum(rows.sum);
        if (!sees) // (a query of zeros, whose sums may have overflowed)
        {
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
                rows.out[d] = zero16();
        }
        store_row<T, DP, Whole>(a.o + n * a.os.sample + head * a.os.head + i * a.os.token, a.dim, rows.out, 1.0f / (sees ? sum : 1.0f));
        if (a.logsumexp && lane < 32)
            a.logsumexp[(static_cast<int64_t>(n) * a.query_heads + head) * a.masks.queries + i] =
                sees ? (rows.max + log2f(sum)) * kLn2 : -INFINITY;
    }
#endif
}

// Few workgroups' worth of queries: the queries of all heads that share a key head are rows one after another, 32 of them a workgroup, so
// that keys and values are read once for them.  The waves of a workgroup go through different tiles of the same part of the keys,
// each with LDS of its own and without barriers, and join what they have at the end.
template <typename T, int DP, int DQ, bool Whole>
__global__ void __launch_bounds__(kThreads) attention_split_kernel(const Args<T> a)
{
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int KT = kTileKeys<T>;
    using Load = TileLoad<T, DP, KT, kWaveSize, Whole>;
    // Tiles that go straight to LDS have a place for keys and one for values; those that pass through registers take turns at one.
    constexpr int kBytes = kTileBytes<T, DP, KT>, kTilesBytes = kWaves * (Load::kDirect ? 2 : 1) * kBytes;
    constexpr int kJoinStride = DP + 4, kJoinBytes = kWaves * kRows * kJoinStride * 4;
    __shared__ __attribute__((aligned(16))) char lds[kTilesBytes > kJoinBytes ? kTilesBytes : kJoinBytes];
    __shared__ float max_sum[kWaves][kRows][2];
    const Place place = place_of(a.order, blockIdx.x, gridDim.x, a.heads, a.query_blocks * a.parts.num);
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
    int from = 0, to = 0;
    if (first_query <= last_query)
    {
        from = sample.first_key(first_query);
        to = sample.end_key(last_query);
    }
    const int tiles = (max(to - from, 0) + KT - 1) / KT;
    const int first_tile = static_cast<int>(static_cast<int64_t>(tiles) * part / a.parts.num);
    const int end_tile = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / a.parts.num);

    const T* const k = a.k + n * a.ks.sample + key_head * a.ks.head;
    const T* const v = a.v + n * a.vs.sample + key_head * a.vs.head;
    const LdsBytes k_tile = (LdsBytes) (lds + wave * (Load::kDirect ? 2 : 1) * kBytes), v_tile = k_tile + (Load::kDirect ? kBytes : 0);
    Load k_load, v_load;
    const auto issue = [&](Load* load, const T* p, const Strides& s, int tile, LdsBytes lds_tile) {
        const int at = from + tile * KT;
        load->issue(buffer_of(p + at * s.token, min(KT, to - at), s.token, a.dim), static_cast<int>(s.token * sizeof(T)),
                    a.dim, lds_tile, lane);
    };

    Rows32<T, DP, DQ> rows;
    rows.clear();
    const bool there = i <= last_query;
    load_fragment<T, DQ, Whole>(&rows.q, a.q + n * a.qs.sample + head * a.qs.head + i * a.qs.token, there, a.dim);
    rows.from = there ? sample.first_key(i) : 0;
    rows.end = there ? sample.end_key(i) : 0;
    const int all_from = sample.first_key(last_query), all_end = sample.end_key(first_query);

    int tile = first_tile + wave;
    if (tile < end_tile)
    {
        issue(&k_load, k, a.ks, tile, k_tile);
        issue(&v_load, v, a.vs, tile, v_tile);
    }
    for (; tile < end_tile; tile += kWaves)
    {
        const int at = from + tile * KT;
        f32x16 s[KT / 32];
        Weights<T> w[KT / 32];
        if constexpr (Load::kDirect)
            wait_for_loads<Load::kEach>(); // the keys are there, the values may be under way
        k_load.put(k_tile, lane);
        rows.score(k_tile, s);
        wait_for_lds();
        const bool more = tile + kWaves < end_tile;
        if (more)
            issue(&k_load, k, a.ks, tile + kWaves, k_tile);
        // (a row beyond the sample's queries sees no key, and its wave no tile as a whole)
        rows.soften(s, w, at, at < all_from || at + KT > all_end, a.scale_log2);
        if constexpr (Load::kDirect)
        {
            if (more)
                wait_for_loads<Load::kEach>();
            else
                wait_for_loads<0>();
        }
        v_load.put(v_tile, lane);
        rows.weigh(v_tile, w);
        wait_for_lds();
        if (more)
            issue(&v_load, v, a.vs, tile + kWaves, v_tile);
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
    const bool sees = my_query < sample.queries && sample.first_key(my_query) < sample.end_key(my_query);
    if (!sees)
        total = 0.0f;
    const int64_t at = (static_cast<int64_t>(n) * a.query_heads + key_head * a.group + my_head) * queries + my_query;
    const int64_t all = static_cast<int64_t>(a.samples) * a.query_heads * queries;
    const bool whole = a.parts.num == 1;
    T* const o = a.o + n * a.os.sample + (key_head * a.group + my_head) * a.os.head + my_query * a.os.token;
    float* const share = a.parts.out + (part * all + at) * DP;
    const float scale = 1.0f / total;
    if (column == 0)
    {
        if (!whole)
        {
            a.parts.max_sum[2 * (part * all + at)] = sees ? max : -INFINITY;
            a.parts.max_sum[2 * (part * all + at) + 1] = total;
        }
        else if (a.logsumexp)
            a.logsumexp[at] = sees ? (max + log2f(total)) * kLn2 : -INFINITY;
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
                o[d + j] = static_cast<T>(sees ? x[j] * scale : 0.0f); // (a query of zeros may have sums that overflowed)
    }
#endif
}

// Joins the parts of a row: a lane has a part's maximum and sum, and S waves (one or four) take every S-th part's output.  (With one wave a
// row, one part after another, 512 rows of 16 parts took 21 us, a chain of waits for memory; with four 16016 rows of two parts 19.)
constexpr int kMostParts = kWaveSize;
template <typename T, int DP, int S>
__global__ void __launch_bounds__(kThreads) attention_join_kernel(const Args<T> a)
{
    constexpr int N = (DP + kWaveSize - 1) / kWaveSize; // elements of a lane
    __shared__ float outs[kWaves][N * kWaveSize], factors[kWaves][kMostParts];
    const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
    const int64_t rows = static_cast<int64_t>(a.samples) * a.query_heads * a.masks.queries;
    const int64_t row = min(static_cast<int64_t>(blockIdx.x) * (kWaves / S) + wave / S, rows - 1); // (the last one more than once)
    float max = kLowest, sum = 0.0f;
    if (lane < a.parts.num)
    {
        max = a.parts.max_sum[2 * (lane * rows + row)];
        sum = a.parts.max_sum[2 * (lane * rows + row) + 1];
    }
    const bool sees = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(max))) > -INFINITY; // (lane 0 has the first part)
    const bool any = !(sum == 0.0f); // (a part without keys counts nothing; one whose sum is NaN makes all NaN)
    const float most = wave_combine(any ? max : kLowest, [](float x, float y) { return fmaxf(x, y); });
    const float factor = any ? __builtin_amdgcn_exp2f(max - most) : 0.0f;
    factors[wave][lane] = factor;
    sum = token::wave_total(sum * factor);
    __syncthreads();
    float out[N] = {};
#pragma unroll 4
    for (int p = wave % S; p < a.parts.num; p += S)
    {
        const float f = factors[wave][p];
#pragma unroll
        for (int n = 0; n < N; ++n)
        {
            const float x = n * kWaveSize + lane < DP ? a.parts.out[(p * rows + row) * DP + n * kWaveSize + lane] : 0.0f;
            out[n] = f != 0.0f ? __builtin_fmaf(x, f, out[n]) : out[n];
        }
    }
    if constexpr (S > 1)
    {
#pragma unroll
        for (int n = 0; n < N; ++n)
            outs[wave][n * kWaveSize + lane] = out[n];
        __syncthreads();
        if (wave > 0)
            return;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int w = 1; w < S; ++w)
                out[n] += outs[w][n * kWaveSize + lane];
    }
    const int64_t of_head = row / a.masks.queries, i = row - of_head * a.masks.queries;
    const int64_t n = of_head / a.query_heads, head = of_head - n * a.query_heads;
    T* const o = a.o + n * a.os.sample + head * a.os.head + i * a.os.token;
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e * kWaveSize + lane < a.dim)
            o[e * kWaveSize + lane] = static_cast<T>(sees ? out[e] / sum : 0.0f);
    if (a.logsumexp && lane == 0)
        a.logsumexp[row] = sees ? (most + log2f(sum)) * kLn2 : -INFINITY;
}

// ---- host ------------------------------------------------------------------------------------------------------

// How a call is run.
struct Plan
{
    bool split; // the keys among the waves of a workgroup
    int query_blocks, parts, padded_dim;
    uint64_t groups; // workgroups
};

Plan plan_of(const h2x_attention& a)
{
    Plan p{};
    const int64_t units = chip_units(), group = a.query_heads / a.key_heads;
    const int64_t wide_blocks = (a.queries + kWaves * kRows - 1) / (kWaves * kRows), wide = wide_blocks * a.samples * a.query_heads;
    const int64_t blocks = (group * a.queries + kRows - 1) / kRows, groups = blocks * a.samples * a.key_heads;
    // Workgroups of 128 queries where there are enough of them: from half a workgroup for each CU on, or where the keys are a tile or two.  (us,
    // 128 queries against split keys, bf16 unless said: 24 such workgroups, 196 keys, 8.8 and 7.5; 80, 577 keys, 13.4 and 11.6; 128, 2048
    // keys, 43.9 and 42.9, causal 41.8 and 30.5; floats, 1001 keys, causal, 82 and 50; 240, 577 keys, 18 and 42; 256, 2048 keys, 48 and 81;
    // 64 and 128, 128 and 64 keys, 6.7 and 7.2, 5.1 and 7.4.)
    p.split = a.queries <= 16 || (2 * wide <= units && a.keys > 128);
    p.padded_dim = (a.head_dim + 31) / 32 * 32;
    p.query_blocks = static_cast<int>(p.split ? blocks : wide_blocks);
    p.parts = 1;
    if (p.split)
    {
        // The keys in parts too while that makes no more workgroups than run at once (twice as many where they are of unlike lengths), 512 keys a
        // part at least; two parts are worth the joining from 4096 keys on.  (us for 1, 2, 4 ... 64 parts: 8 workgroups, 16384 keys of 128, 118,
        // 67, 40, 27, 22, 24, 36; 128 workgroups, 16384 keys, 213, 191, 194, 205; 2048 keys, 27, 30, 35.)
        const bool unlike = a.queries > 16 && (a.window_left < 0) != (a.window_right < 0);
        while (p.parts < kMostParts && groups * p.parts * 2 <= (unlike ? 2 : 1) * units && a.keys >= 1024 * static_cast<int64_t>(p.parts))
            p.parts *= 2;
        if (p.parts == 2 && a.keys < 4096 && !unlike)
            p.parts = 1;
    }
    p.groups = static_cast<uint64_t>(p.split ? groups : wide) * p.parts;
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
        constexpr int DP = decltype(dim)::in_lds, DQ = decltype(dim)::contracted;
        if (p.split)
            launch(attention_split_kernel<T, DP, DQ, Whole>, grid, dim3(kThreads), stream, a);
        else
            launch(attention_forward_kernel<T, DP, DQ, Whole>, grid, dim3(kThreads), stream, a);
        if (p.parts > 4)
            launch(attention_join_kernel<T, DP, 4>, dim3(static_cast<uint32_t>(rows_of(c))), dim3(kThreads), stream, a);
        else if (p.parts > 1)
            launch(attention_join_kernel<T, DP, 1>, dim3(static_cast<uint32_t>((rows_of(c) + kWaves - 1) / kWaves)), dim3(kThreads),
                   stream, a);
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
    if (!q || !o || (c.keys > 0 && (!k || !v || o == k || o == v)) || (p.parts > 1 && !workspace))
        return H2X_ERR_INVALID_ARGUMENT;
    if (o == q && (os.sample != qs.sample || os.token != qs.token || os.head != qs.head)) // (a workgroup overwrites the rows that it has read, and no others)
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
        a.heads = c.samples * (p.split ? c.key_heads : c.query_heads);
        a.order = order_of(c, false);
        return issue<T, decltype(is_whole)::value>(c, p, a, as_stream(stream));
    });
}
