// What the attention kernels share: products of 32 x 32 tiles on the matrix units, tiles in LDS, masks.
//
// All kernels are built alike.  A wave owns 32 rows (queries, or keys where gradients of keys are made), which lie
// along the columns of its matrix tiles: lane l has row l % 32, the two halves of the wave different elements of the
// contracted dimension.  Tiles of the other side pass through LDS, shared by the workgroup.  With the other side as the
// first operand, a tile of scores comes out with a lane's 16 numbers in its own row: sums and maxima along a row are made in
// the lane (and once across the halves), and the probabilities are the second operand of the next product as they lie.
// That product contracts over the other side's rows, so its first operand is the same tile in LDS read across, by the
// transposing LDS loads.
//
// Products are of 16-bit numbers, summed in 32 bits.  Probabilities, and what the backward pass makes of them, are rounded to 16 bits as operands beside
// elements of 16 bits: half a step of theirs for twice the rate at least; sums of probabilities are of those before the rounding.  A float
// is three of them, each the rounding of what those before it leave: eight bits each,
// all 24 (from 2^-109 on, below which the third is no normal number).  Of the nine products of two floats the six that may reach 2^-17 of the
// largest are made; the other three are together at most 2^-24 of it, half a step of a float, and 2^-34.  Six products of 16-bit numbers take three eighths of the time of one by the matrix units' 32-bit
// form.
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

#ifdef __HIPCC__

struct Place
{
    int head, block; // the head counted through all samples
};
// Of workgroup `id` of a grid of `grid`; heads from `heads` on have nothing to do.
__device__ __forceinline__ Place place_of(Order order, uint32_t id, uint32_t grid, uint32_t heads, uint32_t blocks)
{
    if (order == kByHead)
    {
        id = xcd_contiguous(id, grid);
        const uint32_t head = id / blocks;
        return {static_cast<int>(head), static_cast<int>(id - head * blocks)};
    }
    const uint32_t block = id / heads;
    const uint32_t at = id - block * heads;
    if (block >= blocks)
        return {static_cast<int>(heads), 0};
    // workgroups of heads next to each other on one XCD, where the number of heads allows it
    const uint32_t head = heads % kNumXcd == 0 ? at % kNumXcd * (heads / kNumXcd) + at / kNumXcd : at;
    return {static_cast<int>(head), static_cast<int>(order == kFirstFirst ? block : blocks - 1 - block)};
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
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

// ---- elements ------------------------------------------------------------------------------------------------
template <typename T>
constexpr int kPlanes = sizeof(T) == 2 ? 1 : 3; // 16-bit numbers of an element

// x and y as sums of 16-bit numbers, largest first, two numbers to a word as they lie in memory.
__device__ __forceinline__ void split(float x, float y, uint32_t (&v)[3])
{
#pragma unroll
    for (int p = 0; p < 3; ++p)
    {
        v[p] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), bf16x2));
        if (p < 2)
        {
            x -= __uint_as_float(v[p] << 16);
            y -= __uint_as_float(v[p] & 0xffff0000u);
        }
    }
}

// Eight neighbouring elements as they come from memory.
template <typename T>
struct Eight;
template <>
struct Eight<bf16>
{
    u32x4 v;
};
template <>
struct Eight<float>
{
    u32x4 v[2];
};
__device__ __forceinline__ void planes_of(const Eight<bf16>& e, bf16x8 (&out)[1])
{
    out[0] = __builtin_bit_cast(bf16x8, e.v);
}
__device__ __forceinline__ void planes_of(const Eight<float>& e, bf16x8 (&out)[3])
{
    u32x4 words[3];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        uint32_t parts[3];
        split(__uint_as_float(e.v[i / 2][i % 2 * 2]), __uint_as_float(e.v[i / 2][i % 2 * 2 + 1]), parts);
#pragma unroll
        for (int p = 0; p < 3; ++p)
            words[p][i] = parts[p];
    }
#pragma unroll
    for (int p = 0; p < 3; ++p)
        out[p] = __builtin_bit_cast(bf16x8, words[p]);
}
__device__ __forceinline__ float element(const Eight<bf16>& e, int i)
{
    return static_cast<float>(__builtin_bit_cast(bf16x8, e.v)[i]);
}
__device__ __forceinline__ float element(const Eight<float>& e, int i)
{
    return __uint_as_float(e.v[i / 4][i % 4]);
}

// Elements at .. at + 7 of the row at p; zero from dim on, and where the row is not `there`.
template <typename T, bool Whole>
__device__ __forceinline__ Eight<T> load_eight(const T* p, int at, bool there, int dim)
{
    constexpr int N = 16 / sizeof(T);
    u32x4 v[8 / N];
#pragma unroll
    for (int n = 0; n < 8 / N; ++n, at += N)
    {
        v[n] = u32x4{0, 0, 0, 0};
        if constexpr (Whole)
        {
            if (there && at < dim)
                v[n] = *reinterpret_cast<const u32x4*>(p + at);
        }
        else
        {
            AVec<T, N> x;
#pragma unroll
            for (int i = 0; i < N; ++i)
                x.v[i] = there && at + i < dim ? p[at + i] : static_cast<T>(0.0f);
            v[n] = __builtin_bit_cast(u32x4, x);
        }
    }
    return __builtin_bit_cast(Eight<T>, v);
}

// ---- tiles in LDS ------------------------------------------------------------------------------------------
// A tile of R rows of DP 16-bit numbers, in 16-byte chunks; of floats three such, one behind the other.  Chunks are moved about within their row
// so that both ways of reading find their lanes' data on different banks: 16 rows at the same chunk (16 bytes a lane), and 4 rows (row % 4 =
// 0 .. 3) at 4 neighbouring chunks (8 bytes a lane).
template <int DP>
struct Tile
{
    static constexpr int kRowBytes = DP * 2, kChunks = DP / 8;

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
        else
            return chunk ^ (((row & 3) << 2) | ((row >> 2) & 3));
    }
    // The chunk that lies at a place.
    __device__ static __forceinline__ int chunk_at(int row, int at)
    {
        if constexpr (kRowBytes == 192)
        {
            const int chunk = at - ((row >> 2) & 3);
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
template <typename T, int DP, int R>
constexpr int kTileBytes = kPlanes<T>* R* Tile<DP>::kRowBytes;

// A buffer of `rows` rows of `dim` elements, `stride` elements apart: reads behind it give zero.  (The words of a buffer descriptor, the same in all
// lanes.)
template <typename T>
__device__ __forceinline__ u32x4 buffer_of(const T* p, int rows, int64_t stride, int dim)
{
    const int64_t bytes = rows > 0 ? ((rows - 1) * stride + dim) * static_cast<int64_t>(sizeof(T)) : 0;
    const uint64_t base = reinterpret_cast<uint64_t>(p);
    return {static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(base))),
            static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(base >> 32 & 0xffff))),
            static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bytes))), 0x00020000u};
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource_of(const u32x4& b)
{
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(static_cast<uint64_t>(b[1]) << 32 | b[0]), 0, static_cast<int>(b[2]),
                                             static_cast<int>(b[3]));
}
constexpr unsigned int kOutside = 0x80000000u; // behind every buffer

// 16 or 4 bytes a lane from a buffer straight to LDS, to `to` (the same in all lanes) and on.  In assembly, because the compiler waits for
// all loads that its own form of these has issued before it reads any LDS across, those for the next tile among them (gradients of keys,
// heads of 128: 674 us, 550 without loads).  Nothing is returned to registers; who reads the LDS waits with wait_for_loads().  (Five wait states
// between a lane's number put into a scalar register and a load that uses it, one after m0: the compiler does not see to that in assembly.)
// m0 is named as written, so that the compiler keeps no number of its own there from before to behind; it warns that it saves none either.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int Bytes>
__device__ __forceinline__ void load_to_lds(const u32x4& b, unsigned int at, LdsBytes to)
{
    const int place = __builtin_amdgcn_readfirstlane(static_cast<int>(reinterpret_cast<uintptr_t>(to)));
    if constexpr (Bytes == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(place), "v"(at), "s"(b) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(place), "v"(at), "s"(b) : "memory", "m0");
}

#pragma clang diagnostic pop

// Until no more than N of this wave's loads are under way (they arrive in order).
template <int N = 0>
__device__ __forceinline__ void wait_for_loads()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | N >> 4 << 14); // (an instruction that the compiler counts with)
    asm volatile("" ::: "memory");
}
// Until what this wave has asked of LDS is there.
__device__ __forceinline__ void wait_for_lds()
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// How Threads threads (t: this one's number among them) bring R rows of a buffer into a tile.  Whole chunks of 16-bit elements go
// straight to LDS, and are there when the wave that has issued the loads has waited for them; others are held in registers until they are put there.
template <typename T, int DP, int R, int Threads, bool Whole>
struct TileLoad
{
    static constexpr bool kDirect = Whole && sizeof(T) == 2;
    static constexpr int kUnits = R * Tile<DP>::kChunks, kEach = (kUnits + Threads - 1) / Threads; // of eight elements
    static_assert(kUnits % kWaveSize == 0, "whole waves");
    Eight<T> held[kDirect ? 1 : kEach];

    __device__ __forceinline__ void issue(const u32x4& buffer, int stride_bytes, int dim, LdsBytes tile, int t)
    {
        const __amdgpu_buffer_rsrc_t b = resource_of(buffer);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
        {
            const int p = i * Threads + t, of_wave = i * Threads + (t & ~(kWaveSize - 1));
            if (kUnits % Threads != 0 && of_wave >= kUnits)
                break;
            const int row = p / Tile<DP>::kChunks, at = 8 * Tile<DP>::chunk_at(row, p % Tile<DP>::kChunks);
            const unsigned int byte = row * stride_bytes + at * static_cast<int>(sizeof(T));
            if constexpr (kDirect)
                load_to_lds<16>(buffer, at < dim ? byte : kOutside, tile + of_wave * 16);
            else if constexpr (Whole)
            {
                held[i].v[0] = __builtin_amdgcn_raw_buffer_load_b128(b, at < dim ? byte : kOutside, 0, 0);
                held[i].v[1] = __builtin_amdgcn_raw_buffer_load_b128(b, at + 4 < dim ? byte + 16 : kOutside, 0, 0);
            }
            else if constexpr (sizeof(T) == 4)
            {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    held[i].v[j / 4][j % 4] = __builtin_amdgcn_raw_buffer_load_b32(b, at + j < dim ? byte + 4 * j : kOutside, 0, 0);
            }
            else
            {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    const unsigned int lo = static_cast<unsigned short>(
                        __builtin_amdgcn_raw_buffer_load_b16(b, at + 2 * j < dim ? byte + 4 * j : kOutside, 0, 0));
                    const unsigned int hi = static_cast<unsigned short>(
                        __builtin_amdgcn_raw_buffer_load_b16(b, at + 2 * j + 1 < dim ? byte + 4 * j + 2 : kOutside, 0, 0));
                    held[i].v[j] = lo | hi << 16;
                }
            }
        }
    }

    // (The tile is there for other waves after a barrier.)
    __device__ __forceinline__ void put(LdsBytes tile, int t) const
    {
        if constexpr (!kDirect)
        {
#pragma unroll
            for (int i = 0; i < kEach; ++i)
            {
                if (kUnits % Threads != 0 && i * Threads + (t & ~(kWaveSize - 1)) >= kUnits)
                    break;
                bf16x8 planes[kPlanes<T>];
                planes_of(held[i], planes);
#pragma unroll
                for (int p = 0; p < kPlanes<T>; ++p)
                    *reinterpret_cast<__attribute__((address_space(3))) bf16x8*>(tile + (p * kUnits + i * Threads + t) * 16) = planes[p];
            }
        }
    }
};

// ---- products --------------------------------------------------------------------------------------------------
// A row's elements as second operand: what lane l has of row l % 32, for the contraction over DQ elements (a multiple of 16; tiles in LDS have a
// multiple of 32, DP).
template <typename T, int DQ>
struct Fragment
{
    bf16x8 chunk[DQ / 16][kPlanes<T>]; // elements 16 c + 8 (lane / 32) and on
};

// Of the row at p; zero where it is not `there`.
template <typename T, int DQ, bool Whole>
__device__ __forceinline__ void load_fragment(Fragment<T, DQ>* f, const T* p, bool there, int dim)
{
    const int half = (threadIdx.x & (kWaveSize - 1)) / 32;
#pragma unroll
    for (int c = 0; c < DQ / 16; ++c)
        planes_of(load_eight<T, Whole>(p, 16 * c + 8 * half, there, dim), f->chunk[c]);
}

__device__ __forceinline__ f32x16 zero16()
{
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        z[i] = 0.0f;
    return z;
}

__device__ __forceinline__ void multiply(const bf16x8 (&a)[1], const bf16x8 (&b)[1], f32x16* s)
{
    *s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], *s, 0, 0, 0);
}
__device__ __forceinline__ void multiply(const bf16x8 (&a)[3], const bf16x8 (&b)[3], f32x16* s)
{
    *s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2], b[0], *s, 0, 0, 0); // (small ones first)
    *s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[2], *s, 0, 0, 0);
    *s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[1], *s, 0, 0, 0);
    *s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[0], *s, 0, 0, 0);
    *s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[1], *s, 0, 0, 0);
    *s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], *s, 0, 0, 0);
}

// Order of Steps steps, each of Reads reads from LDS and Products products: reads run Ahead steps ahead.  (Left to itself the compiler reads
// into the same registers at each step, and a wave waits for LDS before every product.)
template <int Steps, int Reads, int Products, int Ahead = 6>
__device__ __forceinline__ void read_ahead()
{
    constexpr int kAhead = Ahead < Steps ? Ahead : Steps, kRead = 0x100, kProduct = 0x8;
    __builtin_amdgcn_sched_group_barrier(kRead, kAhead * Reads, 0);
#pragma unroll
    for (int i = 0; i < Steps - kAhead; ++i)
    {
        __builtin_amdgcn_sched_group_barrier(kProduct, Products, 0);
        __builtin_amdgcn_sched_group_barrier(kRead, Reads, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kProduct, kAhead * Products, 0);
}
template <typename T>
constexpr int kProducts = kPlanes<T> == 1 ? 1 : 6; // of two elements

// s[b] (m, n) = sum over DQ of tile[first_row + 32 b + m] * row n of the fragment, of a tile of R rows: lane l's number i has n = l % 32 and
// m = 8 (i / 4) + 4 (l / 32) + i % 4.  (The blocks' chains of products are interleaved: none waits for its own last one.)
template <typename T, int DP, int DQ, int R, int B>
__device__ __forceinline__ void products(LdsBytes tile, int first_row, const Fragment<T, DQ>& f, f32x16 (&s)[B])
{
    using L = Tile<DP>;
    const int lane = threadIdx.x & (kWaveSize - 1);
    const int base = L::address(lane & 31, lane / 32);
#pragma unroll
    for (int b = 0; b < B; ++b)
        s[b] = zero16();
#pragma unroll
    for (int c = 0; c < DQ / 16; ++c)
#pragma unroll
        for (int b = 0; b < B; ++b)
        {
            const LdsBytes at = tile + (first_row + 32 * b) * L::kRowBytes
                                + (L::kFlips ? base ^ 32 * c : L::address(lane & 31, 2 * c + lane / 32));
            bf16x8 a[kPlanes<T>];
#pragma unroll
            for (int p = 0; p < kPlanes<T>; ++p)
                a[p] = *reinterpret_cast<__attribute__((address_space(3))) bf16x8*>(at + p * R * L::kRowBytes);
            multiply(a, f.chunk[c], &s[b]);
        }
    read_ahead<DQ / 16 * B, kPlanes<T>, kProducts<T>>();
}
// 32 x 32 numbers as they come out of products(), as second operand of a contraction over m.
template <typename T>
struct Weights
{
    u32x4 words[2][kPlanes<T>];
    // Numbers i (even) and i + 1 of the lane.
    __device__ __forceinline__ void set(int i, float x, float y)
    {
        if constexpr (kPlanes<T> == 1)
            words[i / 8][0][i % 8 / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), bf16x2));
        else
        {
            uint32_t parts[3];
            split(x, y, parts);
#pragma unroll
            for (int p = 0; p < 3; ++p)
                words[i / 8][p][i % 8 / 2] = parts[p];
        }
    }
    __device__ __forceinline__ void operand(int t, bf16x8 (&v)[kPlanes<T>]) const
    {
#pragma unroll
        for (int p = 0; p < kPlanes<T>; ++p)
            v[p] = __builtin_bit_cast(bf16x8, words[t][p]);
    }
};

// out[d] (e, n) += sum over m of tile[first_row + m][32 d + e] * w(m, n), for the DP / 32 blocks of elements.
template <typename T, int DP, int R>
__device__ __forceinline__ void accumulate(LdsBytes tile, int first_row, const Weights<T>& w, f32x16 (&out)[DP / 32])
{
    using L = Tile<DP>;
    const int lane = threadIdx.x & (kWaveSize - 1);
    // Number i of half h is row 8 (i / 4) + 4 h + i % 4: eight of them, as one operand holds, are two runs of four rows.  A
    // transposing load gives 16 lanes 16 columns of four rows, lane j having loaded four columns of row j / 4.
    const int row = 4 * (lane / 32) + (lane & 15) / 4;
    const int chunk = (lane & 16) / 8 + (lane & 3) / 2, byte = (lane & 1) * 8;
    const int base = L::address(row, chunk) + byte;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int t = 0; t < 2; ++t)
        {
            bf16x8 a[kPlanes<T>], b[kPlanes<T>];
            w.operand(t, b);
#pragma unroll
            for (int p = 0; p < kPlanes<T>; ++p)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                {
                    const LdsBytes at =
                        tile + (p * R + first_row + 16 * t + 8 * u) * L::kRowBytes
                        + (L::kFlips ? base ^ (64 * d + 32 * u) // (rows 8 further on are moved by two chunks more)
                                     : row * L::kRowBytes + L::place(16 * t + 8 * u + row, 4 * d + chunk) * 16 + byte);
                    const bf16x4 part = __builtin_bit_cast(
                        bf16x4,
                        __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4*>(at)));
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        a[p][4 * u + i] = part[i];
                }
            multiply(a, b, &out[d]);
        }
    read_ahead<DP / 16, 2 * kPlanes<T>, kProducts<T>>();
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
    if (!(a->scale >= 1e-30) || !(a->scale <= 1e30)) // (in 32 bits neither zero, which an infinite score would make NaN, nor infinite)
        return H2X_ERR_INVALID_ARGUMENT;
    if (a->head_dim > 128)
        return H2X_ERR_UNSUPPORTED;
    const int64_t heads = a->query_heads > 0 ? a->query_heads : a->key_heads; // (query heads are no fewer where there are any)
    if (a->queries > 0x7fffffff - 256 || a->keys > 0x7fffffff - 256 || a->samples * heads > 0x7fffffff)
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
// tiles: the longest first, so that the short ones fill up the end.
inline Order order_of(const h2x_attention& a, bool keys)
{
    const bool left = a.window_left >= 0, right = a.window_right >= 0;
    return left == right ? kByHead : right != keys ? kLastFirst : kFirstFirst;
}

// Elements of a head in LDS, a multiple of 32, and in a contraction, of 16.
template <int P, int Q>
struct Padded
{
    static constexpr int in_lds = P, contracted = Q;
};
// f(Padded()) for heads of `dim` elements.
template <typename F>
int with_padded_dim(int dim, const F& f)
{
    return dim <= 32   ? f(Padded<32, 32>())
           : dim <= 64 ? f(Padded<64, 64>())
           : dim <= 80 ? f(Padded<96, 80>()) // (72 and 80 are common; a sixth of two products)
           : dim <= 96 ? f(Padded<96, 96>())
                       : f(Padded<128, 128>());
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
