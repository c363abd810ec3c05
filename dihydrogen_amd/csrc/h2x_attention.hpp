// What the attention kernels share: products of 32 x 32 tiles on the matrix units, tiles in LDS, masks.
//
// All kernels are built alike.  A wave owns 32 rows (queries, or keys where gradients of keys are made), which lie
// along the columns of its matrix tiles: lane l has row l % 32, the two halves of the wave different elements of the
// contracted dimension.  Tiles of the other side pass through LDS, shared by the workgroup.  With the other side as the
// first operand, a tile of scores comes out with a lane's 16 numbers in its own row: sums and maxima along a row are made in
// the lane (and once across the halves), and the probabilities are the second operand of the next product as they lie.
// That product contracts over the other side's rows, so its first operand is the same tile in LDS read across:
// 16-bit elements by the transposing LDS loads, 32-bit ones singly.
#pragma once

#include "h2x_token.hpp"

// (Kernels that use buffers have no body on the host, whose compiler does not know their type.)

namespace h2x
{
namespace attention
{

using token::bf16;

constexpr int kRows = 32; // of a wave
constexpr int kThreads = 256, kWaves = kThreads / kWaveSize;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;
constexpr int64_t kMostTokenStride = 1 << 21; // 128 rows of 4-byte elements span less than 2^31 bytes

using Strides = h2x_token_strides;

struct Masks
{
    const int32_t *query_lengths, *key_lengths;
    int32_t queries, keys;
    int32_t left, right; // largest int32: no bound
};

// A sample's lengths, and where its queries stand among its keys.
struct Sample
{
    int32_t queries, keys;
    int32_t left, right;

    // Keys that query i sees: [first_key(i), end_key(i)), both within [0, keys] and growing with i.
    __host__ __device__ int32_t first_key(int64_t i) const
    {
        const int64_t at = i + keys - queries - left;
        return static_cast<int32_t>(at < 0 ? 0 : at < keys ? at : keys);
    }
    __host__ __device__ int32_t end_key(int64_t i) const
    {
        const int64_t at = i + keys - queries + right + 1;
        return static_cast<int32_t>(at < 0 ? 0 : at < keys ? at : keys);
    }
    // Queries that see key j.
    __host__ __device__ int32_t first_query(int64_t j) const
    {
        const int64_t at = j - keys + queries - right;
        return static_cast<int32_t>(at < 0 ? 0 : at < queries ? at : queries);
    }
    __host__ __device__ int32_t end_query(int64_t j) const
    {
        const int64_t at = j - keys + queries + left + 1;
        return static_cast<int32_t>(at < 0 ? 0 : at < queries ? at : queries);
    }
};

// In which order workgroups go through the blocks of rows of all heads (of all samples).
enum Order
{
    kByHead,     // head after head, each XCD a run of them: heads' keys and values stay in its L2
    kFirstFirst, // the first blocks of all heads, which have the most to do, then the second ones ...
    kLastFirst   // the same from the last ones on
};
struct Schedule
{
    Order order;
    int fold; // blocks from this one on come the other way round
};

#ifdef __HIPCC__

struct Place
{
    int head, block; // the head counted through all samples
};
// Of workgroup `id` of a grid of `grid`; heads from `heads` on have nothing to do.
__device__ __forceinline__ Place place_of(const Schedule& s, uint32_t id, uint32_t grid, uint32_t heads, uint32_t blocks)
{
    if (s.order == kByHead)
    {
        id = xcd_contiguous(id, grid);
        const uint32_t head = id / blocks;
        return {static_cast<int>(head), static_cast<int>(id - head * blocks)};
    }
    uint32_t block = id / heads;
    const uint32_t at = id - block * heads;
    if (block >= blocks)
        return {static_cast<int>(heads), 0};
    if (block >= static_cast<uint32_t>(s.fold))
        block = s.fold + blocks - 1 - block;
    // workgroups of heads next to each other on one XCD, where the number of heads allows it
    const uint32_t head = heads % kNumXcd == 0 ? at % kNumXcd * (heads / kNumXcd) + at / kNumXcd : at;
    return {static_cast<int>(head), static_cast<int>(s.order == kFirstFirst ? block : blocks - 1 - block)};
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
using LdsBytes = __attribute__((address_space(3))) char*;

__device__ __forceinline__ int32_t clamp_length(int32_t n, int32_t most)
{
    return n < 0 ? 0 : n < most ? n : most;
}
__device__ __forceinline__ Sample sample_of(const Masks& m, int sample)
{
    return {m.query_lengths ? clamp_length(m.query_lengths[sample], m.queries) : m.queries,
            m.key_lengths ? clamp_length(m.key_lengths[sample], m.keys) : m.keys, m.left, m.right};
}

// What the other half of the wave has for the same row, combined with one's own.
__device__ __forceinline__ float halves_max(float v)
{
    return combine_apart<32>(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float halves_sum(float v)
{
    return combine_apart<32>(v, [](float a, float b) { return a + b; });
}

// ---- tiles in LDS ------------------------------------------------------------------------------------------
// A tile of rows of DP elements, in 16-byte chunks.  Chunks are moved about within their row so that both ways of reading
// find their lanes' data on different banks: 16 rows at the same chunk (16 bytes a lane), and 4 rows (row % 4 = 0 .. 3) at
// 4 neighbouring chunks (8 bytes a lane).
template <typename T, int DP>
struct Tile
{
    static constexpr int kRowBytes = DP * sizeof(T), kChunks = kRowBytes / 16, kPerChunk = 16 / sizeof(T);

    __device__ static __forceinline__ int place(int row, int chunk)
    {
        if constexpr (kRowBytes == 64)
            return chunk ^ ((row >> 2) & 3);
        else if constexpr (kRowBytes == 128)
            return chunk ^ (((row & 2) << 1) | ((row >> 2) & 3));
        else if constexpr (kRowBytes == 192)
        {
            const int at = chunk + ((row >> 2) & 3);
            return at >= kChunks ? at - kChunks : at;
        }
        else if constexpr (kRowBytes == 256)
            return chunk ^ (((row & 3) << 2) | ((row >> 2) & 3));
        else if constexpr (kRowBytes == 384)
        {
            const int at = chunk + ((row >> 1) & 7);
            return at >= kChunks ? at - kChunks : at;
        }
        else
            return chunk ^ (row & 15);
    }
    // The chunk that lies at a place.
    __device__ static __forceinline__ int chunk_at(int row, int at)
    {
        if constexpr (kRowBytes == 192)
        {
            const int chunk = at - ((row >> 2) & 3);
            return chunk < 0 ? chunk + kChunks : chunk;
        }
        else if constexpr (kRowBytes == 384)
        {
            const int chunk = at - ((row >> 1) & 7);
            return chunk < 0 ? chunk + kChunks : chunk;
        }
        else
            return place(row, at);
    }
    __device__ static __forceinline__ int address(int row, int chunk)
    {
        return row * kRowBytes + place(row, chunk) * 16;
    }
    // Rows whose chunks are moved by exclusive or: so are addresses, by what chunk numbers differ in.
    static constexpr bool kFlips = (kRowBytes & (kRowBytes - 1)) == 0;
};

// A number that the compiler does not know: what is worked out from it is worked out where it is used, and not kept in registers from
// one round of a loop to the next.
template <bool Lean>
__device__ __forceinline__ int once(int v)
{
    if constexpr (Lean)
        asm volatile("" : "+v"(v));
    return v;
}

// A buffer of `rows` rows of `dim` elements, `stride` elements apart: reads behind it give zero.
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const T* p, int rows, int64_t stride, int dim)
{
    const int64_t bytes = rows > 0 ? ((rows - 1) * stride + dim) * static_cast<int64_t>(sizeof(T)) : 0;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, static_cast<int>(bytes), 0x00020000);
}
constexpr unsigned int kOutside = 0x80000000u; // behind every buffer

// One 16-byte chunk of a row that may begin on any element.
template <typename T>
__device__ __forceinline__ u32x4 load_elements(__amdgpu_buffer_rsrc_t b, int row, int chunk, int stride_bytes, int dim)
{
    constexpr int N = 16 / sizeof(T);
    const unsigned int at = row * stride_bytes + chunk * 16;
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        if constexpr (sizeof(T) == 4)
            v[i] = __builtin_amdgcn_raw_buffer_load_b32(b, chunk * N + i < dim ? at + 4 * i : kOutside, 0, 0);
        else
        {
            const unsigned int lo = static_cast<unsigned short>(
                __builtin_amdgcn_raw_buffer_load_b16(b, chunk * N + 2 * i < dim ? at + 4 * i : kOutside, 0, 0));
            const unsigned int hi = static_cast<unsigned short>(
                __builtin_amdgcn_raw_buffer_load_b16(b, chunk * N + 2 * i + 1 < dim ? at + 4 * i + 2 : kOutside, 0, 0));
            v[i] = lo | hi << 16;
        }
    }
    return v;
}

// Loads R rows of a buffer into a tile, by Threads threads (t: this one's number among them).  Whole chunks go straight to LDS, and
// are there when the wave that loads them has waited for its loads; others through registers, and are there after a barrier.
template <typename T, int DP, int R, int Threads, bool Whole>
__device__ __forceinline__ void load_tile(__amdgpu_buffer_rsrc_t b, int stride_bytes, int dim, LdsBytes tile, int t)
{
    using L = Tile<T, DP>;
    constexpr int kTotal = R * L::kChunks;
    static_assert(kTotal % kWaveSize == 0, "whole waves");
#pragma unroll
    for (int i = 0; i < kTotal; i += Threads)
    {
        const int p = i + t;
        if (kTotal % Threads != 0 && i + (t & ~(kWaveSize - 1)) >= kTotal)
            break;
        const int row = p / L::kChunks, chunk = L::chunk_at(row, p % L::kChunks);
        if constexpr (Whole)
        {
            const unsigned int at = row * stride_bytes + chunk * 16;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                b, reinterpret_cast<__attribute__((address_space(3))) void*>(tile + (i + (t & ~(kWaveSize - 1))) * 16), 16,
                chunk * L::kPerChunk < dim ? at : kOutside, 0, 0, 0);
        }
        else
            *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(tile + p * 16) =
                load_elements<T>(b, row, chunk, stride_bytes, dim);
    }
}

// 64 numbers of a buffer to LDS, by a wave.
__device__ __forceinline__ void load_numbers(__amdgpu_buffer_rsrc_t b, LdsBytes to, int lane)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, reinterpret_cast<__attribute__((address_space(3))) void*>(to), 4, lane * 4, 0, 0, 0);
}

// Until no more than N of this wave's loads are under way (they arrive in order).
template <int N = 0>
__device__ __forceinline__ void wait_for_loads()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Until what this wave has asked of LDS is there.
__device__ __forceinline__ void wait_for_lds()
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// ---- products --------------------------------------------------------------------------------------------------
// A row's elements as second operand: what lane l has of row l % 32, for the contraction over DP elements.
template <typename T, int DP>
struct Fragment
{
    u32x4 chunk[Tile<T, DP>::kChunks / 2]; // chunks 2 c + (lane / 32)
};

// Of the row at p; zero where it is not `there`.
template <typename T, int DP, bool Whole>
__device__ __forceinline__ void load_fragment(Fragment<T, DP>* f, const T* p, bool there, int dim)
{
    constexpr int N = 16 / sizeof(T);
    const int half = (threadIdx.x & (kWaveSize - 1)) / 32;
#pragma unroll
    for (int c = 0; c < Tile<T, DP>::kChunks / 2; ++c)
    {
        const int at = (2 * c + half) * N;
        u32x4 v = {0, 0, 0, 0};
        if constexpr (Whole)
        {
            if (there && at < dim)
                v = *reinterpret_cast<const u32x4*>(p + at);
        }
        else
        {
            AVec<T, N> x;
#pragma unroll
            for (int i = 0; i < N; ++i)
                x.v[i] = there && at + i < dim ? p[at + i] : static_cast<T>(0.0f);
            v = __builtin_bit_cast(u32x4, x);
        }
        f->chunk[c] = v;
    }
}

__device__ __forceinline__ f32x16 zero16()
{
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        z[i] = 0.0f;
    return z;
}

// s[b] (m, n) = sum over DP of tile[first_row + 32 b + m] * row n of the fragment: lane l's number i has n = l % 32 and
// m = 8 (i / 4) + 4 (l / 32) + i % 4.  (The blocks' chains of products are interleaved: none waits for its own last one.)
template <typename T, int DP, int B, bool Lean = false>
__device__ __forceinline__ void products(LdsBytes tile, int first_row, const Fragment<T, DP>& f, f32x16 (&s)[B])
{
    using L = Tile<T, DP>;
    const int lane = threadIdx.x & (kWaveSize - 1);
    const int base = once<Lean>(L::address(lane & 31, lane / 32));
#pragma unroll
    for (int b = 0; b < B; ++b)
        s[b] = zero16();
#pragma unroll
    for (int c = 0; c < L::kChunks / 2; ++c)
#pragma unroll
        for (int b = 0; b < B; ++b)
        {
            const LdsBytes at = tile + (first_row + 32 * b) * L::kRowBytes
                                + (L::kFlips ? base ^ 32 * c : L::address(lane & 31, 2 * c + lane / 32));
            if constexpr (sizeof(T) == 2)
            {
                const bf16x8 a = *reinterpret_cast<__attribute__((address_space(3))) bf16x8*>(at);
                s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, f.chunk[c]), s[b], 0, 0, 0);
            }
            else
            {
                const f32x4 a = *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(at);
                const f32x4 w = __builtin_bit_cast(f32x4, f.chunk[c]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], w[i], s[b], 0, 0, 0);
            }
        }
}
template <typename T, int DP, bool Lean = false>
__device__ __forceinline__ f32x16 product(LdsBytes tile, int first_row, const Fragment<T, DP>& f)
{
    f32x16 s[1];
    products<T, DP, 1, Lean>(tile, first_row, f, s);
    return s[0];
}

// The same of two tiles' rows with a fragment each, 32 rows: s from the first, t from the second.
template <typename T, int DP, bool Lean = false>
__device__ __forceinline__ void two_products(LdsBytes tile_s, LdsBytes tile_t, int first_row, const Fragment<T, DP>& f,
                                             const Fragment<T, DP>& g, f32x16* s, f32x16* t)
{
    using L = Tile<T, DP>;
    const int lane = threadIdx.x & (kWaveSize - 1);
    const int base = once<Lean>(L::address(lane & 31, lane / 32));
    *s = zero16();
    *t = zero16();
#pragma unroll
    for (int c = 0; c < L::kChunks / 2; ++c)
    {
        const int at = first_row * L::kRowBytes + (L::kFlips ? base ^ 32 * c : L::address(lane & 31, 2 * c + lane / 32));
        if constexpr (sizeof(T) == 2)
        {
            const bf16x8 a = *reinterpret_cast<__attribute__((address_space(3))) bf16x8*>(tile_s + at);
            const bf16x8 b = *reinterpret_cast<__attribute__((address_space(3))) bf16x8*>(tile_t + at);
            *s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, f.chunk[c]), *s, 0, 0, 0);
            *t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b, __builtin_bit_cast(bf16x8, g.chunk[c]), *t, 0, 0, 0);
        }
        else
        {
            const f32x4 a = *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(tile_s + at);
            const f32x4 b = *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(tile_t + at);
            const f32x4 u = __builtin_bit_cast(f32x4, f.chunk[c]), v = __builtin_bit_cast(f32x4, g.chunk[c]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                *s = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], u[i], *s, 0, 0, 0);
                *t = __builtin_amdgcn_mfma_f32_32x32x2f32(b[i], v[i], *t, 0, 0, 0);
            }
        }
    }
}

// 32 x 32 numbers as they come out of products(), as second operand of a contraction over m.
template <typename T>
struct Weights;
template <>
struct Weights<bf16>
{
    bf16x8 v[2];
    __device__ __forceinline__ void set(int i, float x) { v[i / 8][i % 8] = static_cast<bf16>(x); }
};
template <>
struct Weights<float>
{
    float v[16];
    __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
};

// out[d] (e, n) += sum over m of tile[first_row + m][32 d + e] * w(m, n), for the DP / 32 blocks of elements.
template <int DP, bool Lean = false>
__device__ __forceinline__ void accumulate(LdsBytes tile, int first_row, const Weights<bf16>& w, f32x16 (&out)[DP / 32])
{
    using L = Tile<bf16, DP>;
    const int lane = threadIdx.x & (kWaveSize - 1);
    // Number i of half h is row 8 (i / 4) + 4 h + i % 4: eight of them, as one operand holds, are two runs of four rows.  A
    // transposing load gives 16 lanes 16 columns of four rows, lane j having loaded four columns of row j / 4.
    const int row = 4 * (lane / 32) + (lane & 15) / 4;
    const int chunk = (lane & 16) / 8 + (lane & 3) / 2, byte = (lane & 1) * 8;
    const int base = once<Lean>(L::address(row, chunk) + byte);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int t = 0; t < 2; ++t)
        {
            bf16x8 a;
#pragma unroll
            for (int u = 0; u < 2; ++u)
            {
                const LdsBytes at =
                    tile + (first_row + 16 * t + 8 * u) * L::kRowBytes
                    + (L::kFlips ? base ^ (64 * d + 32 * u) // (rows 8 further on are moved by two chunks more)
                                 : row * L::kRowBytes + L::place(16 * t + 8 * u + row, 4 * d + chunk) * 16 + byte);
                const bf16x4 part = __builtin_bit_cast(
                    bf16x4,
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4*>(at)));
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    a[4 * u + i] = part[i];
            }
            out[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, w.v[t], out[d], 0, 0, 0);
        }
}
template <int DP, bool Lean = false>
__device__ __forceinline__ void accumulate(LdsBytes tile, int first_row, const Weights<float>& w, f32x16 (&out)[DP / 32])
{
    using L = Tile<float, DP>;
    const int lane = threadIdx.x & (kWaveSize - 1);
#pragma unroll
    for (int i = 0; i < 16; ++i)
    {
        const int row = 8 * (i / 4) + i % 4 + 4 * (lane / 32);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
        {
            const float a = *reinterpret_cast<__attribute__((address_space(3))) float*>(
                tile + first_row * L::kRowBytes + L::address(row, 8 * d + (lane & 31) / 4) + (lane & 3) * 4);
            out[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w.v[i], out[d], 0, 0, 0);
        }
    }
}

// Stores what accumulate() made of row l % 32 (v times factor), at p; Whole: rows begin on multiples of 16 bytes.
template <typename T, int DP, bool Whole>
__device__ __forceinline__ void store_row(T* p, int dim, const f32x16 (&v)[DP / 32], float factor)
{
    const int half = (threadIdx.x & (kWaveSize - 1)) / 32;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
        {
            const int at = 32 * d + 2 * i + 4 * half;
            if constexpr (Whole)
            {
                if (at < dim)
                {
                    AVec<T, 4> x;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x.v[j] = static_cast<T>(v[d][i + j] * factor);
                    *reinterpret_cast<AVec<T, 4>*>(p + at) = x;
                }
            }
            else
            {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at + j < dim)
                        p[at + j] = static_cast<T>(v[d][i + j] * factor);
            }
        }
}

// The scores of 32 rows of a tile (rows first .. first + 31 on its side) that a lane's row does not see become -infinity: it sees
// [from, end).
__device__ __forceinline__ void hide(f32x16* s, int first, int from, int end)
{
    asm volatile(""); // (most tiles are seen as a whole: a branch, no work that is thrown away)
    const int half = (threadIdx.x & (kWaveSize - 1)) / 32;
    const unsigned int seen = end > from ? end - from : 0;
    const int at = first + 4 * half - from;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        (*s)[i] = static_cast<unsigned int>(at + 8 * (i / 4) + i % 4) < seen ? (*s)[i] : -INFINITY;
}

#endif // __HIPCC__

// ---- host ------------------------------------------------------------------------------------------------------

// What both directions check.
inline int check(const h2x_attention* a)
{
    if (!a)
        return H2X_ERR_INVALID_ARGUMENT;
    if (a->dtype != H2X_BF16 && a->dtype != H2X_F32)
        return H2X_ERR_UNSUPPORTED;
    if (a->head_dim < 1 || a->samples < 0 || a->query_heads < 0 || a->key_heads < 0 || a->queries < 0 || a->keys < 0
        || (a->query_heads > 0 && (a->key_heads < 1 || a->query_heads % a->key_heads != 0)))
        return H2X_ERR_INVALID_ARGUMENT;
    if (!(a->scale > 0) || !(a->scale <= 1e30))
        return H2X_ERR_INVALID_ARGUMENT;
    if (a->head_dim > 128)
        return H2X_ERR_UNSUPPORTED;
    if (a->queries > 0x7fffffff - 256 || a->keys > 0x7fffffff - 256)
        return H2X_ERR_TOO_LARGE;
    return H2X_SUCCESS;
}

// The strides of a tensor of so many samples, tokens and heads: one that no element depends on is zero.
inline Strides strides_of(const h2x_attention& a, const h2x_token_strides& s, int64_t tokens, int heads)
{
    return {a.samples > 1 ? s.sample : 0, tokens > 1 ? s.token : 0, heads > 1 ? s.head : 0};
}

// Tokens lie apart and not too far; in an output samples and heads do not lie on one another either.
inline int check_strides(const h2x_attention& a, const Strides& s, int64_t tokens, int heads, bool output)
{
    if (tokens > 1 && s.token < a.head_dim)
        return H2X_ERR_INVALID_ARGUMENT;
    if (output && ((a.samples > 1 && s.sample < a.head_dim) || (heads > 1 && s.head < a.head_dim)))
        return H2X_ERR_INVALID_ARGUMENT;
    return s.token > kMostTokenStride ? H2X_ERR_UNSUPPORTED : H2X_SUCCESS;
}

// Whether all rows of a tensor are whole 16-byte chunks.
inline bool whole_rows(const h2x_attention& a, const void* p, const Strides& s)
{
    const int n = a.dtype == H2X_F32 ? 4 : 8;
    return a.head_dim % n == 0 && aligned16(p) && s.sample % n == 0 && s.token % n == 0 && s.head % n == 0;
}

inline Masks masks_of(const h2x_attention& a, const int32_t* query_lengths, const int32_t* key_lengths)
{
    const auto bound = [](int64_t w) { return static_cast<int32_t>(w < 0 || w > 0x7fffffff ? 0x7fffffff : w); };
    return {query_lengths,
            key_lengths,
            static_cast<int32_t>(a.queries),
            static_cast<int32_t>(a.keys),
            bound(a.window_left),
            bound(a.window_right)};
}

// The order for blocks of queries, or of keys, which are the other way round.  Under a mask that bounds one side blocks have unlike numbers of
// tiles: the longest first, so that the short ones fill up the end.  Where all workgroups run at once, two a CU, the second one of a CU is the
// shorter the longer its first.
inline Schedule schedule_of(const h2x_attention& a, bool keys, uint64_t heads, uint64_t blocks)
{
    const bool left = a.window_left >= 0, right = a.window_right >= 0;
    if (left == right)
        return {kByHead, 0};
    return {right != keys ? kLastFirst : kFirstFirst, static_cast<int>(blocks)};
}

// f(std::integral_constant<int, DP>) for heads padded to a multiple of 32 elements.
template <typename F>
int with_padded_dim(int dim, const F& f)
{
    return dim <= 32   ? f(std::integral_constant<int, 32>())
           : dim <= 64 ? f(std::integral_constant<int, 64>())
           : dim <= 96 ? f(std::integral_constant<int, 96>())
                       : f(std::integral_constant<int, 128>());
}

// f(T(), Whole) for the type of the elements.
template <typename F>
int with_elements(int dtype, bool whole, const F& f)
{
    if (dtype == H2X_F32)
        return whole ? f(float(), std::true_type()) : f(float(), std::false_type());
    return whole ? f(bf16(), std::true_type()) : f(bf16(), std::false_type());
}

} // namespace attention
} // namespace h2x
