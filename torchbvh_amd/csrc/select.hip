// Choice of key blocks: for every block of queries the `count` blocks of its
// cloud whose boxes are nearest to the centre of the queries' box.
//
//   centre_a = 0.5 lo_a + 0.5 hi_a  over the block's queries (NaNs left out)
//   d_a = max(lo'_a - centre_a, centre_a - hi'_a, 0),  score = d_0^2 + d_1^2 (+ d_2^2)
//
// in fp32, in that order and without fused multiply-adds, so a choice is
// reproducible bit for bit; ties go to the lower block number, and blocks whose
// score is not finite are not chosen.
#include "attend.hpp"

namespace tbvh {
namespace {

constexpr uint64_t kNoBlock = ~uint64_t{0};

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int src) {
    return static_cast<uint64_t>(__shfl(static_cast<unsigned long long>(v), src, kWave));
}

// The cloud of block `b`: the last one whose first block is at most b.  The
// lanes look at 64 clouds at a time.
__device__ __forceinline__ int cloud_of(const int64_t* __restrict__ firsts, int clouds, int64_t b) {
    int before = 0;
    for (int i = 0; i < clouds; i += kWave) {
        const int c = i + lane_id();
        before += __popcll(__ballot(c < clouds && firsts[c] <= b));
    }
    return before - 1;
}

template <int D>
__device__ __forceinline__ float box_score(const float* __restrict__ box, const float (&centre)[D]) {
    float score = 0.0f;
    bool bad = false;
#pragma unroll
    for (int x = 0; x < D; ++x) {
        const float below = box[x] - centre[x], above = centre[x] - box[D + x];
        const float d = fmaxf(fmaxf(below, above), 0.0f);
        bad |= below != below || above != above;
        score = x == 0 ? d * d : score + d * d;
    }
    return bad ? INFINITY : score;
}

// One wave per block of queries.  Lane i holds the i-th best key so far, a key
// being (score, block) in 64 bits; 64 boxes are scored at a time and those
// that beat the last kept key are put in their places one by one.
template <int D>
__global__ __launch_bounds__(kWave) void select_kernel(SelectArgs a) {
    const int lane = lane_id();
    const int64_t group = blockIdx.x;
    const Rows rows = block_rows(a.q_starts, group, a.q_block, a.q_total);
    float lo[D], hi[D], centre[D];
#pragma unroll
    for (int x = 0; x < D; ++x) {
        lo[x] = INFINITY;
        hi[x] = -INFINITY;
    }
    for (int i = lane; i < rows.count; i += kWave) {
#pragma unroll
        for (int x = 0; x < D; ++x) {
            const float v = a.queries[(rows.first + i) * D + x];
            lo[x] = fminf(lo[x], v);
            hi[x] = fmaxf(hi[x], v);
        }
    }
#pragma unroll
    for (int x = 0; x < D; ++x) centre[x] = 0.5f * wave_min(lo[x]) + 0.5f * wave_max(hi[x]);

    const int cloud = cloud_of(a.q_clouds, a.clouds, group);
    const int64_t first = cloud < 0 ? 0 : max(a.k_clouds[cloud], int64_t{0});
    const int64_t last = cloud < 0 ? 0 : min(a.k_clouds[cloud + 1], static_cast<int64_t>(a.blocks));
    uint64_t best = kNoBlock, limit = kNoBlock;
    for (int64_t b0 = first; b0 < last; b0 += kWave) {
        const int64_t b = b0 + lane;
        uint64_t key = kNoBlock;
        if (b < last) {
            const float score = box_score<D>(a.boxes + b * 2 * D, centre);
            if (score < INFINITY) key = static_cast<uint64_t>(__float_as_uint(score)) << 32 | static_cast<uint32_t>(b);
        }
        for (uint64_t todo = __ballot(key < limit); todo != 0; todo &= todo - 1) {
            const uint64_t x = shfl64(key, __builtin_ctzll(todo));
            if (x >= limit) continue;
            const int at = __popcll(__ballot(best < x));
            const uint64_t up = shfl64(best, lane > 0 ? lane - 1 : 0);
            best = lane < at ? best : lane == at ? x : up;
            limit = shfl64(best, a.count - 1);
        }
    }
    if (lane < a.count) a.out[group * a.count + lane] = best == kNoBlock ? -1 : static_cast<int32_t>(best);
}

}  // namespace

hipError_t launch_select(const SelectArgs& a, int D, hipStream_t stream) {
    if (a.groups == 0) return hipSuccess;
    if (D == 2) select_kernel<2><<<a.groups, kWave, 0, stream>>>(a);
    else select_kernel<3><<<a.groups, kWave, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace tbvh
