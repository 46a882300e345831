// Attention over chosen blocks, forward (the formulas and the tiles' layout
// are in attend.hpp).
#include "attend.hpp"

namespace tbvh {
namespace {

constexpr int kChunk = 64;  // keys per step of the running softmax

// One work-group of W waves per (row block, key head, tile of RT * 16 rows of
// the block's queries times the heads that share the key head); wave w takes
// every W-th chosen block, and the waves' parts are joined at the end.
// DP: channels padded to a multiple of 32.
template <typename T, int DP, int RT, int W, bool kBias>
__global__ __launch_bounds__(kWave* W) void attend_kernel(AttendArgs a, int tiles, int64_t items) {
    constexpr int DS = DP / 32, DT = DP / 16, KT = kChunk / 16;
    constexpr int LDV = DP + 16 / sizeof(T);  // LDS row stride
    extern __shared__ float4 s_raw[];
    const int lane = lane_id(), n = lane & 15, g = lane >> 4;
    const int wave = W == 1 ? 0 : threadIdx.x / kWave;
    const int64_t item = xcd_item(blockIdx.x, gridDim.x);
    if (item >= items) return;
    const int c = static_cast<int>(item % a.kv_heads);
    const int64_t tile_item = item / a.kv_heads;
    const int tile = static_cast<int>(tile_item % tiles);
    const int64_t group = tile_item / tiles;
    const Rows qr = block_rows(a.q_starts, group, a.q_block, a.q_total);
    const int rows = qr.count * a.share;
    if (tile * RT * 16 >= rows) return;

    T* s_v = reinterpret_cast<T*>(s_raw) + wave * kChunk * LDV;
    float* s_bias = reinterpret_cast<float*>(reinterpret_cast<T*>(s_raw) + W * kChunk * LDV);
    const int span = 2 * a.reach + 1, entries = a.axes * span;
    if constexpr (kBias) {
        const T* table = static_cast<const T*>(a.table);
        for (int i = threadIdx.x; i < a.share * entries; i += kWave * W) {
            const int hs = i / entries, e = i - hs * entries, axis = e / span;
            const int b = min(max(a.map[e - axis * span], 0), a.buckets - 1);
            s_bias[i] = static_cast<float>(table[(axis * a.buckets + b) * a.heads + c * a.share + hs]) * kLog2e;
        }
        __syncthreads();
    }

    Vec8<T> qf[RT][DS];
    int qc[RT][3];
    const float* bias_row[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int rr = tile * RT * 16 + rt * 16 + n;
        const bool real = rr < rows;
        const int qi = real ? rr / a.share : 0, hs = real ? rr - qi * a.share : 0;
        const T* row = static_cast<const T*>(a.q) + (qr.first + qi) * a.q_row + (c * a.share + hs) * a.q_head;
#pragma unroll
        for (int s = 0; s < DS; ++s) qf[rt][s] = load8(row, 32 * s + 8 * g, a.D, real);
        if constexpr (kBias) {
            bias_row[rt] = s_bias + hs * entries;
#pragma unroll
            for (int x = 0; x < 3; ++x) qc[rt][x] = x < a.axes ? a.q_cells[(qr.first + qi) * a.axes + x] : 0;
        }
    }

    f32x4 acc[RT][DT];
    float top[RT], sum[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        top[rt] = -INFINITY;
        sum[rt] = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[rt][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const float to_log2 = a.scale * kLog2e;

    for (int slot = wave; slot < a.count; slot += W) {
        const int block = __builtin_amdgcn_readfirstlane(a.selected[group * a.count + slot]);
        if (block < 0 || block >= a.blocks) continue;
        const Rows kr = block_rows(a.k_starts, block, a.k_block, a.k_total);
        for (int base = 0; base < kr.count; base += kChunk) {
            const T* k0 = static_cast<const T*>(a.k) + (kr.first + base) * a.k_row + c * a.k_head;
            const T* v0 = static_cast<const T*>(a.v) + (kr.first + base) * a.v_row + c * a.v_head;
            const int left = kr.count - base;
            wave_sync();
#pragma unroll
            for (int i = 0; i < DP / 8; ++i) {
                const int p = lane + kWave * i, row = p / (DP / 8), d = p % (DP / 8) * 8;
                *reinterpret_cast<Vec8<T>*>(s_v + row * LDV + d) = load8(v0 + row * a.v_row, d, a.D, row < left);
            }
            f32x4 st[KT][RT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                Vec8<T> kf[DS];
                const int row = 16 * kt + n;
#pragma unroll
                for (int s = 0; s < DS; ++s) kf[s] = load8(k0 + row * a.k_row, 32 * s + 8 * g, a.D, row < left);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int s = 0; s < DS; ++s) x = mma(kf[s], qf[rt][s], x);
                    st[kt][rt] = x * to_log2;
                }
                if constexpr (kBias) {
                    for (int x = 0; x < a.axes; ++x) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int key = min(16 * kt + 4 * g + r, left - 1);
                            const int kc = a.k_cells[(kr.first + base + key) * a.axes + x];
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
                                const int q = x == 0 ? qc[rt][0] : x == 1 ? qc[rt][1] : qc[rt][2];
                                st[kt][rt][r] += bias_row[rt][x * span + cell_offset(q, kc, a.reach)];
                            }
                        }
                    }
                }
                if (left < kChunk) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (16 * kt + 4 * g + r >= left)
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) st[kt][rt][r] = -INFINITY;
                }
            }
            Vec8<T> pf[KT / 2][RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float m = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) m = fmaxf(m, st[kt][rt][r]);
                m = fmaxf(top[rt], across_groups_max(m));
                // Rows that have met no finite score yet keep weights of zero.
                const float ref = m == -INFINITY ? 0.0f : m;
                const float keep = __builtin_amdgcn_exp2f(top[rt] - ref);
                top[rt] = m;
                float part = 0.0f;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        st[kt][rt][r] = __builtin_amdgcn_exp2f(st[kt][rt][r] - ref);
                        part += st[kt][rt][r];
                    }
                sum[rt] = sum[rt] * keep + part;
#pragma unroll
                for (int t = 0; t < DT; ++t) acc[rt][t] *= keep;
                // Weights are rounded to T for the product with v (2^-9 each in
                // bf16, independent); their sum is kept in fp32.
#pragma unroll
                for (int p = 0; p < KT / 2; ++p) pf[p][rt] = join<T>(st[2 * p][rt], st[2 * p + 1][rt]);
            }
            wave_sync();
#pragma unroll
            for (int p = 0; p < KT / 2; ++p)
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    Vec8<T> vf;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        vf[j] = s_v[(32 * p + 16 * (j / 4) + 4 * g + j % 4) * LDV + 16 * t + n];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) acc[rt][t] = mma(vf, pf[p][rt], acc[rt][t]);
                }
        }
    }

#pragma unroll
    for (int rt = 0; rt < RT; ++rt) sum[rt] = across_groups_sum(sum[rt]);
    if constexpr (W > 1) {
        // Every wave's (top, sum, acc) through LDS; wave 0 joins them in order.
        float* s_part = reinterpret_cast<float*>(s_raw);
        constexpr int kPer = RT * (DT * 4 + 2) * kWave;
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float* p = s_part + wave * kPer + rt * (DT * 4 + 2) * kWave + lane;
            p[0] = top[rt];
            p[kWave] = sum[rt];
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) p[(2 + t * 4 + r) * kWave] = acc[rt][t][r];
        }
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float* p = s_part + rt * (DT * 4 + 2) * kWave + lane;
            float m = top[rt];
            for (int w = 1; w < W; ++w) m = fmaxf(m, p[w * kPer]);
            const float ref = m == -INFINITY ? 0.0f : m;
            const float keep = __builtin_amdgcn_exp2f(top[rt] - ref);
            sum[rt] *= keep;
#pragma unroll
            for (int t = 0; t < DT; ++t) acc[rt][t] *= keep;
            for (int w = 1; w < W; ++w) {
                const float f = __builtin_amdgcn_exp2f(p[w * kPer] - ref);
                sum[rt] += p[w * kPer + kWave] * f;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[rt][t][r] += p[w * kPer + (2 + t * 4 + r) * kWave] * f;
            }
            top[rt] = m;
        }
    }

#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int rr = tile * RT * 16 + rt * 16 + n;
        if (rr >= rows) continue;
        const int qi = rr / a.share, hs = rr - qi * a.share;
        const int64_t at = (qr.first + qi) * a.heads + c * a.share + hs;
        const float inverse = sum[rt] == 0.0f ? 0.0f : 1.0f / sum[rt];
        T* row = static_cast<T*>(a.out) + at * a.D;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            const int d = 16 * t + 4 * g;
            if (d < a.D) {
                Vec4<T> o;
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = static_cast<T>(acc[rt][t][r] * inverse);
                *reinterpret_cast<Vec4<T>*>(row + d) = o;
            }
        }
        // 0 for an empty row: its scores are all -inf, their weights 0 again.
        if (a.lse != nullptr && g == 0) a.lse[at] = sum[rt] == 0.0f ? 0.0f : top[rt] + __builtin_amdgcn_logf(sum[rt]);
    }
}

template <typename T, int DP, int RT, int W>
hipError_t launch(const AttendArgs& a, hipStream_t stream) {
    const int tiles = (a.q_block * a.share + RT * 16 - 1) / (RT * 16);
    const int64_t items = static_cast<int64_t>(a.groups) * tiles * a.kv_heads;
    const unsigned grid = static_cast<unsigned>(xcd_grid(items));
    const size_t stage = static_cast<size_t>(W) * kChunk * (DP + 16 / sizeof(T)) * sizeof(T);
    const size_t bias = static_cast<size_t>(a.share) * a.axes * (2 * a.reach + 1) * sizeof(float);
    const size_t parts = W > 1 ? static_cast<size_t>(W) * RT * (DP / 16 * 4 + 2) * kWave * sizeof(float) : 0;
    if (a.table != nullptr) {
        const auto kernel = attend_kernel<T, DP, RT, W, true>;
        const size_t lds = std::max(stage + bias, parts);
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
        if (e != hipSuccess) return e;
        kernel<<<grid, kWave * W, lds, stream>>>(a, tiles, items);
    } else {
        const auto kernel = attend_kernel<T, DP, RT, W, false>;
        const size_t lds = std::max(stage, parts);
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
        if (e != hipSuccess) return e;
        kernel<<<grid, kWave * W, lds, stream>>>(a, tiles, items);
    }
    return hipGetLastError();
}

// Row tiles: 16 rows where a block has no more, else 64, or 32 where the
// accumulators of 64 would not fit the registers (fp32, more than 64
// channels).  Waves per tile: enough that a call of few tiles covers the chip.
template <typename T, int DP>
hipError_t launch_rows(const AttendArgs& a, hipStream_t stream) {
    constexpr int kWide = sizeof(T) == 2 && DP <= 64 ? 4 : 2;
    const int rows = a.q_block * a.share;
    constexpr int64_t kFill = 2048;  // waves that fill the 256 CUs twice a SIMD
    if (rows <= 16) {
        const int64_t items = static_cast<int64_t>(a.groups) * a.kv_heads;
        // Eight waves' staged values fit the LDS but for fp32 rows of 128.
        constexpr int kMany = sizeof(T) * DP <= 256 ? 8 : 4;
        if (items * 4 <= kFill && a.count > 1) return launch<T, DP, 1, kMany>(a, stream);
        return launch<T, DP, 1, 1>(a, stream);
    }
    const int64_t items = static_cast<int64_t>(a.groups) * ((rows + kWide * 16 - 1) / (kWide * 16)) * a.kv_heads;
    if (items * 2 <= kFill && a.count > 1) return launch<T, DP, kWide, 4>(a, stream);
    return launch<T, DP, kWide, 1>(a, stream);
}

template <typename T>
hipError_t launch_type(const AttendArgs& a, hipStream_t stream) {
    if (a.D <= 32) return launch_rows<T, 32>(a, stream);
    if (a.D <= 64) return launch_rows<T, 64>(a, stream);
    return launch_rows<T, 128>(a, stream);
}

}  // namespace

hipError_t launch_attend(const AttendArgs& a, bool bf16, hipStream_t stream) {
    return bf16 ? launch_type<__bf16>(a, stream) : launch_type<float>(a, stream);
}

}  // namespace tbvh
