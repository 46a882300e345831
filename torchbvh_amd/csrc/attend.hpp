// Attention over chosen blocks: what its forward and backward kernels share.
//
// Rows are packed cloud after cloud and cut into blocks; row block g of the
// queries attends to the keys of the blocks selected[g, 0..m).  With head h of
// the queries reading head h / share of the keys,
//
//   s_ij = scale q_i . k_j + sum_a table[a, bucket(cq_ia - ck_ja), h]
//   o_i  = sum_j exp(s_ij - lse_i) v_j,   lse_i = log sum_j exp(s_ij).
//
// Products run on 16 x 16 MFMA tiles with fp32 accumulators.  A fragment is
// 8 values a lane along the contraction: lane (i = lane % 16, g = lane / 16)
// holds operand row i at depths 8 g .. 8 g + 7 of 32.  In an accumulator lane
// (n, g) holds rows 4 g .. 4 g + 3 of column n.  Scores are computed with the
// axis that the next product contracts along the accumulator's rows, so two
// tiles' accumulators, rounded, are that product's fragment as they stand:
// its depth slot (g, j) then means row 4 g + j of the first tile for j < 4 and
// row 4 g + j - 4 of the second for the others.  Contraction order is free, so
// only the other operand has to be read in the same order (a transposed read).
#pragma once

#include "tbvh_internal.hpp"

namespace tbvh {

using f32x4 = float __attribute__((ext_vector_type(4)));
using f32x8 = float __attribute__((ext_vector_type(8)));
using bf16x4 = __bf16 __attribute__((ext_vector_type(4)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));

template <typename T>
struct Pack;
template <>
struct Pack<float> {
    using V4 = f32x4;
    using V8 = f32x8;
};
template <>
struct Pack<__bf16> {
    using V4 = bf16x4;
    using V8 = bf16x8;
};
template <typename T>
using Vec4 = typename Pack<T>::V4;
template <typename T>
using Vec8 = typename Pack<T>::V8;

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// Depth 32 in eight products of depth 4: step j takes slot j of every group.
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// Eight channels from channel d of a row; zeros past D (a multiple of 8).
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* __restrict__ row, int d, int D, bool real) {
    Vec8<T> v = {};
    if (real && d < D) v = *reinterpret_cast<const Vec8<T>*>(row + d);
    return v;
}

template <typename T>
__device__ __forceinline__ Vec8<T> join(f32x4 a, f32x4 b) {
    Vec8<T> v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = static_cast<T>(a[j]);
        v[4 + j] = static_cast<T>(b[j]);
    }
    return v;
}

// Rows of a packed block: [first, first + count), never past the tensor.
struct Rows {
    int64_t first;
    int count;
};
__device__ __forceinline__ Rows block_rows(const int64_t* __restrict__ starts, int64_t b, int block, int64_t total) {
    const int64_t lo = min(max(starts[b], int64_t{0}), total);
    const int64_t hi = min(max(starts[b + 1], lo), total);
    return {lo, static_cast<int>(min(hi - lo, static_cast<int64_t>(block)))};
}

struct AttendArgs {
    const void* q = nullptr;
    const void* k = nullptr;
    const void* v = nullptr;
    int64_t q_row = 0, q_head = 0, k_row = 0, k_head = 0, v_row = 0, v_head = 0;  // strides, elements
    const int32_t* selected = nullptr;  // (groups, count)
    const int64_t* q_starts = nullptr;  // (groups + 1)
    const int64_t* k_starts = nullptr;  // (blocks + 1)
    int64_t q_total = 0, k_total = 0;   // rows
    int groups = 0, blocks = 0, count = 0;
    int q_block = 0, k_block = 0;       // rows of a full block
    int heads = 0, kv_heads = 0, share = 1, D = 0;
    float scale = 1.0f;
    // Bias: table (axes, buckets, heads), map (2 reach + 1), cells (rows, axes).
    const void* table = nullptr;
    const int32_t* map = nullptr;
    const int32_t* q_cells = nullptr;
    const int32_t* k_cells = nullptr;
    int axes = 0, buckets = 0, reach = 0;
    void* out = nullptr;   // (q_total, heads, D)
    float* lse = nullptr;  // (q_total, heads), base 2; null: not wanted
};

struct AttendGrads {
    const void* grad = nullptr;   // (q_total, heads, D) like out
    float* delta = nullptr;       // (q_total, heads)
    const uint32_t* keys = nullptr;   // sorted block numbers of the (group, slot) entries
    const int64_t* order = nullptr;   // their entries
    const int32_t* runs = nullptr;    // (blocks + 1) first sorted entry of each block
    void* dq = nullptr;           // (q_total, heads, D)
    void* dk = nullptr;           // (k_total, kv_heads, D)
    void* dv = nullptr;
    void* dtable = nullptr;       // like table
    float* table_parts = nullptr; // (parts, heads, axes * buckets)
    int parts = 0;
};

// Bins of the table's gradient that one head may have: each has 64 copies in
// LDS, one a lane, so that no two lanes add to one word and the order of the
// additions is fixed.
constexpr int kMaxBins = 256;
// Entries of one head's table expanded over all distances.
constexpr int kMaxReachEntries = 4096;

// Position of a launch's work-group in its list of items, with consecutive
// items on one XCD: work-groups go to the eight XCDs in turn, and neighbouring
// row blocks choose overlapping key blocks, which that XCD's L2 then holds.
constexpr int kXcds = 8;
__host__ __device__ inline int64_t xcd_grid(int64_t items) { return (items + kXcds - 1) / kXcds * kXcds; }
__device__ __forceinline__ int64_t xcd_item(int64_t block, int64_t grid) {
    return block % kXcds * (grid / kXcds) + block / kXcds;
}

// LDS that the lanes of one wave write and then read from each other: the
// hardware keeps a wave's LDS operations in order, the compiler is told to.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

__device__ __forceinline__ float across_groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float across_groups_sum(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

// Distance of two cells on an axis, clamped to [-reach, reach], from zero up.
__device__ __forceinline__ int cell_offset(int a, int b, int reach) {
    const int d = __builtin_elementwise_sub_sat(a, b);
    return min(max(d, -reach), reach) + reach;
}

hipError_t launch_attend(const AttendArgs& a, bool bf16, hipStream_t stream);
hipError_t launch_attend_backward(const AttendArgs& a, const AttendGrads& g, bool bf16, hipStream_t stream);
// Parts of the table's gradient for these sizes.
int attend_table_parts(int groups, int q_block, int heads);

// Inverse of a selection: the (group, slot) entries sorted by block.
hipError_t launch_invert(const int32_t* selected, int64_t entries, int blocks, Segment* segs, int64_t tiles,
                         const SortBuffers& sb, int64_t* order, int32_t* runs, hipStream_t stream);

struct SelectArgs {
    const float* queries = nullptr;     // (q_total, D)
    const float* boxes = nullptr;       // (blocks, 2 D)
    const int64_t* q_starts = nullptr;
    const int64_t* q_clouds = nullptr;  // (clouds + 1) first group of each cloud
    const int64_t* k_clouds = nullptr;  // (clouds + 1) first block
    int64_t q_total = 0;
    int groups = 0, blocks = 0, clouds = 0, q_block = 0, count = 0;
    float* coarse = nullptr;            // (ceil(blocks / 64), 2 D) boxes of 64 blocks each
    int32_t* out = nullptr;             // (groups, count)
};
hipError_t launch_select(const SelectArgs& a, int D, hipStream_t stream);

}  // namespace tbvh
