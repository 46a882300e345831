// Attention over chosen blocks, backward (formulas and tile layout in
// attend.hpp).  With p = exp2(s - lse) recomputed from the scores,
//
//   dp_ij = grad_i . v_j,  delta_i = grad_i . o_i,  ds_ij = p_ij (dp_ij - delta_i)
//   dq_i = scale sum_j ds_ij k_j     dk_j = scale sum_i ds_ij q_i
//   dv_j = sum_i p_ij grad_i         dtable[a, b, h] = sum of ds_ij over bucket_a(ij) = b.
//
// Two kernels: one owns query rows (dq, delta, the table), one owns key rows and
// visits the row blocks that chose them, found by sorting the selection by block.
// No sum is left to atomics, so every call gives the same bits.
#include "attend.hpp"

namespace tbvh {
namespace {

constexpr int kStep = 32;  // rows of the other side per step

// Work-groups of the query-side kernel with a bias: each takes many tiles of one
// head, so that few parts of the table's gradient are left to add up.
constexpr int kTableParts = 192;  // per head, at most

// One wave per (tile of RT * 16 rows of a row block, head), or, with a bias, per
// list of them: tiles part, part + parts, ... of one head.
template <typename T, int DP, int RT, bool kBias>
__global__ __launch_bounds__(kWave) void attend_dq_kernel(AttendArgs a, AttendGrads gr, int tiles, int64_t items) {
    constexpr int DS = DP / 32, DT = DP / 16, KT = kStep / 16;
    constexpr int LD = DP + 16 / sizeof(T);
    extern __shared__ float4 s_raw[];
    const int lane = lane_id(), n = lane & 15, g = lane >> 4;
    const int64_t item = xcd_item(blockIdx.x, gridDim.x);
    if (item >= items) return;
    const int h = static_cast<int>(item % a.heads), c = h / a.share;
    const int64_t first = item / a.heads;
    const int64_t all_tiles = static_cast<int64_t>(a.groups) * tiles;

    T* s_k = reinterpret_cast<T*>(s_raw);
    float* s_bias = reinterpret_cast<float*>(s_k + kStep * LD);
    const int span = 2 * a.reach + 1, entries = a.axes * span, bins = a.axes * a.buckets;
    int* s_bin = reinterpret_cast<int*>(s_bias + entries);
    float* s_sum = reinterpret_cast<float*>(s_bin + entries);  // (bins, 64): a copy a lane
    if constexpr (kBias) {
        const T* table = static_cast<const T*>(a.table);
        for (int e = lane; e < entries; e += kWave) {
            const int axis = e / span;
            const int bin = axis * a.buckets + min(max(a.map[e - axis * span], 0), a.buckets - 1);
            s_bias[e] = static_cast<float>(table[bin * a.heads + h]) * kLog2e;
            s_bin[e] = bin * kWave;
        }
        for (int i = 0; i < bins; ++i) s_sum[i * kWave + lane] = 0.0f;
        wave_sync();
    }
    const float to_log2 = a.scale * kLog2e;

    for (int64_t at = first; at < all_tiles; at += kBias ? gr.parts : all_tiles) {
        const int tile = static_cast<int>(at % tiles);
        const int64_t group = at / tiles;
        const Rows qr = block_rows(a.q_starts, group, a.q_block, a.q_total);
        if (tile * RT * 16 >= qr.count) continue;
        Vec8<T> qf[RT][DS], gf[RT][DS];
        int qc[RT][3];
        float lse[RT], delta[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int rr = tile * RT * 16 + rt * 16 + n;
            const bool real = rr < qr.count;
            const int64_t row = qr.first + (real ? rr : 0);
            const T* qrow = static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head;
            const T* grow = static_cast<const T*>(gr.grad) + (row * a.heads + h) * a.D;
            const T* orow = static_cast<const T*>(a.out) + (row * a.heads + h) * a.D;
            float dot = 0.0f;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                qf[rt][s] = load8(qrow, 32 * s + 8 * g, a.D, real);
                gf[rt][s] = load8(grow, 32 * s + 8 * g, a.D, real);
                const Vec8<T> o = load8(orow, 32 * s + 8 * g, a.D, real);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    dot = __builtin_fmaf(static_cast<float>(gf[rt][s][j]), static_cast<float>(o[j]), dot);
            }
            delta[rt] = across_groups_sum(dot);
            lse[rt] = a.lse[row * a.heads + h];
            if (real && g == 0) gr.delta[row * a.heads + h] = delta[rt];
            if constexpr (kBias) {
#pragma unroll
                for (int x = 0; x < 3; ++x) qc[rt][x] = x < a.axes ? cell_bytes(a.q_cells[row * a.axes + x]) : 0;
            }
        }
        f32x4 acc[RT][DT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < DT; ++t) acc[rt][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

        for (int slot = 0; slot < a.count; ++slot) {
            const int block = __builtin_amdgcn_readfirstlane(a.selected[group * a.count + slot]);
            if (block < 0 || block >= a.blocks) continue;
            const Rows kr = block_rows(a.k_starts, block, a.k_block, a.k_total);
            for (int base = 0; base < kr.count; base += kStep) {
                const T* k0 = static_cast<const T*>(a.k) + (kr.first + base) * a.k_row + c * a.k_head;
                const T* v0 = static_cast<const T*>(a.v) + (kr.first + base) * a.v_row + c * a.v_head;
                const int left = kr.count - base;
                f32x4 ds[KT][RT];
                wave_sync();
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const int row = 16 * kt + n;
                    Vec8<T> kf[DS], vf[DS];
#pragma unroll
                    for (int s = 0; s < DS; ++s) {
                        kf[s] = load8(k0 + row * a.k_row, 32 * s + 8 * g, a.D, row < left);
                        vf[s] = load8(v0 + row * a.v_row, 32 * s + 8 * g, a.D, row < left);
                        *reinterpret_cast<Vec8<T>*>(s_k + row * LD + 32 * s + 8 * g) = kf[s];
                    }
                    f32x4 st[RT];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int s = 0; s < DS; ++s) x = mma(kf[s], qf[rt][s], x);
                        st[rt] = x * to_log2;
                    }
                    if constexpr (kBias) {
                        for (int x = 0; x < a.axes; ++x) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int key = min(16 * kt + 4 * g + r, left - 1);
                                const int kc = cell_bytes(a.k_cells[(kr.first + base + key) * a.axes + x]);
#pragma unroll
                                for (int rt = 0; rt < RT; ++rt) {
                                    const int q = x == 0 ? qc[rt][0] : x == 1 ? qc[rt][1] : qc[rt][2];
                                    st[rt][r] += s_bias[x * span + a.reach + cell_distance(q, kc, 4 * a.reach) / 4];
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        f32x4 dp = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int s = 0; s < DS; ++s) dp = mma(vf[s], gf[rt][s], dp);
                        const bool real = tile * RT * 16 + rt * 16 + n < qr.count;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float p = __builtin_amdgcn_exp2f(st[rt][r] - lse[rt]);
                            const bool in = real && 16 * kt + 4 * g + r < left;
                            ds[kt][rt][r] = in ? p * (dp[r] - delta[rt]) : 0.0f;
                        }
                    }
                    if constexpr (kBias) {
                        for (int x = 0; x < a.axes; ++x) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int key = min(16 * kt + 4 * g + r, left - 1);
                                const int kc = cell_bytes(a.k_cells[(kr.first + base + key) * a.axes + x]);
#pragma unroll
                                for (int rt = 0; rt < RT; ++rt) {
                                    const int q = x == 0 ? qc[rt][0] : x == 1 ? qc[rt][1] : qc[rt][2];
                                    float* bin = s_sum + s_bin[x * span + a.reach + cell_distance(q, kc, 4 * a.reach) / 4] + lane;
                                    *bin += ds[kt][rt][r];
                                }
                            }
                        }
                    }
                }
                wave_sync();
                // ds is rounded to T for the product with k.
                Vec8<T> df[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) df[rt] = join<T>(ds[0][rt], ds[1][rt]);
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    Vec8<T> kf;
#pragma unroll
                    for (int j = 0; j < 8; ++j) kf[j] = s_k[(16 * (j / 4) + 4 * g + j % 4) * LD + 16 * t + n];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) acc[rt][t] = mma(kf, df[rt], acc[rt][t]);
                }
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int rr = tile * RT * 16 + rt * 16 + n;
            if (rr >= qr.count) continue;
            T* row = static_cast<T*>(gr.dq) + ((qr.first + rr) * a.heads + h) * a.D;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const int d = 16 * t + 4 * g;
                if (d < a.D) {
                    Vec4<T> o;
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = static_cast<T>(acc[rt][t][r] * a.scale);
                    *reinterpret_cast<Vec4<T>*>(row + d) = o;
                }
            }
        }
    }
    if constexpr (kBias) {
        wave_sync();
        float* part = gr.table_parts + (first * a.heads + h) * bins;
        for (int b = lane; b < bins; b += kWave) {
            float total = 0.0f;
            // Lane b starts at its own copy: 64 banks apart from its neighbours'.
            for (int i = 0; i < kWave; ++i) total += s_sum[b * kWave + ((i + b) & (kWave - 1))];
            part[b] = total;
        }
    }
}

// The parts of the table's gradient, in order: one wave per (bin, head).
template <typename T>
__global__ __launch_bounds__(kWave) void table_sum_kernel(const float* __restrict__ parts, int count, int heads, int bins,
                                                          T* __restrict__ out) {
    const int h = blockIdx.x % heads, b = blockIdx.x / heads;
    float total = 0.0f;
    for (int i = lane_id(); i < count; i += kWave) total += parts[(static_cast<int64_t>(i) * heads + h) * bins + b];
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) total += __shfl_xor(total, d, kWave);
    if (lane_id() == 0) out[b * heads + h] = static_cast<T>(total);
}

// One wave per (32 rows of a key block, key head).  The rows of every chosen
// row block's queries, for every head that shares the key head, are taken as one
// list, 32 at a time.
template <typename T, int DP, bool kBias>
__global__ __launch_bounds__(kWave) void attend_dkv_kernel(AttendArgs a, AttendGrads gr, int tiles, int64_t items) {
    constexpr int DS = DP / 32, DT = DP / 16, KT = 2, RT = kStep / 16;
    constexpr int LD = DP + 16 / sizeof(T);
    extern __shared__ float4 s_raw[];
    const int lane = lane_id(), n = lane & 15, g = lane >> 4;
    const int64_t item = xcd_item(blockIdx.x, gridDim.x);
    if (item >= items) return;
    const int c = static_cast<int>(item % a.kv_heads);
    const int tile = static_cast<int>(item / a.kv_heads % tiles);
    const int64_t block = item / a.kv_heads / tiles;
    const Rows kr = block_rows(a.k_starts, block, a.k_block, a.k_total);
    const int base = tile * KT * 16, left = kr.count - base;
    if (left <= 0) return;

    T* s_q = reinterpret_cast<T*>(s_raw);
    T* s_g = s_q + kStep * LD;
    float* s_lse = reinterpret_cast<float*>(s_g + kStep * LD);
    float* s_delta = s_lse + kStep;
    int* s_cell = reinterpret_cast<int*>(s_delta + kStep);  // (3, 32)
    int* s_head = s_cell + 3 * kStep;
    float* s_bias = reinterpret_cast<float*>(s_head + kStep);
    const int span = 2 * a.reach + 1, entries = a.axes * span;
    if constexpr (kBias) {
        const T* table = static_cast<const T*>(a.table);
        for (int i = lane; i < a.share * entries; i += kWave) {
            const int hs = i / entries, e = i - hs * entries, axis = e / span;
            const int b = min(max(a.map[e - axis * span], 0), a.buckets - 1);
            s_bias[i] = static_cast<float>(table[(axis * a.buckets + b) * a.heads + c * a.share + hs]) * kLog2e;
        }
    }
    Vec8<T> kf[KT][DS], vf[KT][DS];
    int kc[KT][3];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int row = 16 * kt + n;
        const bool real = row < left;
        const int64_t at = kr.first + base + (real ? row : 0);
#pragma unroll
        for (int s = 0; s < DS; ++s) {
            kf[kt][s] = load8(static_cast<const T*>(a.k) + at * a.k_row + c * a.k_head, 32 * s + 8 * g, a.D, real);
            vf[kt][s] = load8(static_cast<const T*>(a.v) + at * a.v_row + c * a.v_head, 32 * s + 8 * g, a.D, real);
        }
        if constexpr (kBias) {
#pragma unroll
            for (int x = 0; x < 3; ++x) kc[kt][x] = x < a.axes ? cell_bytes(a.k_cells[at * a.axes + x]) : 0;
        }
    }
    f32x4 dk[KT][DT], dv[KT][DT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int t = 0; t < DT; ++t) dk[kt][t] = dv[kt][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const float to_log2 = a.scale * kLog2e;

    const int run = gr.runs[block];
    const int per = a.q_block * a.share;
    const int64_t list = static_cast<int64_t>(gr.runs[block + 1] - run) * per;
    for (int64_t v0 = 0; v0 < list; v0 += kStep) {
        // Lane l < 32 finds row l of the step and leaves its values in LDS.
        Vec8<T> qf[RT][DS], gf[RT][DS];
        wave_sync();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int64_t v = v0 + 16 * rt + n;
            const int64_t slot = v / per;
            const int rr = static_cast<int>(v - slot * per);
            const int qi = rr / a.share, hs = rr - qi * a.share;
            bool real = v < list;
            int64_t row = 0;
            if (real) {
                const Rows qr = block_rows(a.q_starts, gr.order[run + slot] / a.count, a.q_block, a.q_total);
                real = qi < qr.count;
                row = qr.first + (real ? qi : 0);
            }
            const int h = c * a.share + hs;
            const T* qrow = static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head;
            const T* grow = static_cast<const T*>(gr.grad) + (row * a.heads + h) * a.D;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                qf[rt][s] = load8(qrow, 32 * s + 8 * g, a.D, real);
                gf[rt][s] = load8(grow, 32 * s + 8 * g, a.D, real);
                *reinterpret_cast<Vec8<T>*>(s_q + (16 * rt + n) * LD + 32 * s + 8 * g) = qf[rt][s];
                *reinterpret_cast<Vec8<T>*>(s_g + (16 * rt + n) * LD + 32 * s + 8 * g) = gf[rt][s];
            }
            if (g == 0) {
                // A row that is not there weighs nothing: exp2(s - inf) = 0.
                s_lse[16 * rt + n] = real ? a.lse[row * a.heads + h] : INFINITY;
                s_delta[16 * rt + n] = real ? gr.delta[row * a.heads + h] : 0.0f;
                if constexpr (kBias) {
                    s_head[16 * rt + n] = hs * entries;
                    for (int x = 0; x < a.axes; ++x)
                        s_cell[x * kStep + 16 * rt + n] = real ? cell_bytes(a.q_cells[row * a.axes + x]) : 0;
                }
            }
        }
        wave_sync();
        f32x4 p[RT][KT], ds[RT][KT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const f32x4 lse = *reinterpret_cast<const f32x4*>(s_lse + 16 * rt + 4 * g);
            const f32x4 delta = *reinterpret_cast<const f32x4*>(s_delta + 16 * rt + 4 * g);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f}, dp = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < DS; ++s) {
                    x = mma(qf[rt][s], kf[kt][s], x);
                    dp = mma(gf[rt][s], vf[kt][s], dp);
                }
                x = x * to_log2;
                if constexpr (kBias) {
                    for (int ax = 0; ax < a.axes; ++ax) {
                        const int key = ax == 0 ? kc[kt][0] : ax == 1 ? kc[kt][1] : kc[kt][2];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int q = 16 * rt + 4 * g + r;
                            x[r] += s_bias[s_head[q] + ax * span + a.reach + cell_distance(s_cell[ax * kStep + q], key, 4 * a.reach) / 4];
                        }
                    }
                }
                const bool in = 16 * kt + n < left;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float w = lse[r] == INFINITY || !in ? 0.0f : __builtin_amdgcn_exp2f(x[r] - lse[r]);
                    p[rt][kt][r] = w;
                    ds[rt][kt][r] = lse[r] == INFINITY || !in ? 0.0f : w * (dp[r] - delta[r]);
                }
            }
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            const Vec8<T> pf = join<T>(p[0][kt], p[1][kt]), df = join<T>(ds[0][kt], ds[1][kt]);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                Vec8<T> gt, qt;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int at = (16 * (j / 4) + 4 * g + j % 4) * LD + 16 * t + n;
                    gt[j] = s_g[at];
                    qt[j] = s_q[at];
                }
                dv[kt][t] = mma(gt, pf, dv[kt][t]);
                dk[kt][t] = mma(qt, df, dk[kt][t]);
            }
        }
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        if (16 * kt + n >= left) continue;
        const int64_t at = ((kr.first + base + 16 * kt + n) * a.kv_heads + c) * a.D;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            const int d = 16 * t + 4 * g;
            if (d < a.D) {
                Vec4<T> x, y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = static_cast<T>(dk[kt][t][r] * a.scale);
                    y[r] = static_cast<T>(dv[kt][t][r]);
                }
                *reinterpret_cast<Vec4<T>*>(static_cast<T*>(gr.dk) + at + d) = x;
                *reinterpret_cast<Vec4<T>*>(static_cast<T*>(gr.dv) + at + d) = y;
            }
        }
    }
}

// First launch of the inversion: the sort key of entry e = group * count + slot is
// its block, `blocks` where none is chosen, and every tile counts its first digits.
__global__ __launch_bounds__(kBlock) void invert_keys_kernel(const int32_t* __restrict__ selected, int entries,
                                                             int blocks, Segment* segs, uint32_t* __restrict__ keys,
                                                             uint32_t* __restrict__ tile_hist, int64_t tstride) {
    __shared__ int s_seg;
    __shared__ uint32_t s_cnt[kRadix];
    store_uniform_table(segs, 1, entries, false);
    int seg;
    const Segment g = first_launch_segment(segs, 1, UniformPlan{segs, entries, false}, blockIdx.x, &s_seg, &seg);
    for (int i = threadIdx.x; i < kRadix; i += kBlock) s_cnt[i] = 0u;
    __syncthreads();
    const int lt = static_cast<int>(blockIdx.x - g.tile_first);
    const int count = lt < g.tiles ? min(kSortTile, g.n - lt * kSortTile) : 0;
    for (int i = threadIdx.x; i < count; i += kBlock) {
        const int e = lt * kSortTile + i;
        const int b = selected[e];
        const uint32_t key = static_cast<uint32_t>(b >= 0 && b < blocks ? b : blocks);
        keys[e] = key;
        atomicAdd(&s_cnt[key & (kRadix - 1)], 1u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRadix; i += kBlock) tile_hist[hist_at(i, blockIdx.x, tstride)] = s_cnt[i];
}

// runs[b]: the first sorted entry whose block is b or more.
__global__ __launch_bounds__(kBlock) void invert_runs_kernel(const uint32_t* __restrict__ keys, int entries, int blocks,
                                                             int32_t* __restrict__ runs) {
    const int b = blockIdx.x * kBlock + threadIdx.x;
    if (b > blocks) return;
    int lo = 0, hi = entries;
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (keys[mid] < static_cast<uint32_t>(b)) lo = mid + 1;
        else hi = mid;
    }
    runs[b] = lo;
}

template <typename K>
hipError_t allow_lds(K kernel, size_t bytes) {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(bytes));
}

template <typename T, int DP, int RT, bool kBias>
hipError_t launch_dq(const AttendArgs& a, const AttendGrads& g, hipStream_t stream) {
    const int tiles = (a.q_block + RT * 16 - 1) / (RT * 16);
    const int64_t items = (kBias ? g.parts : static_cast<int64_t>(a.groups) * tiles) * a.heads;
    const int entries = a.axes * (2 * a.reach + 1);
    const size_t lds = kStep * (DP + 16 / sizeof(T)) * sizeof(T) +
                       (kBias ? (entries * 2 + static_cast<size_t>(a.axes) * a.buckets * kWave) * sizeof(float) : 0);
    const auto kernel = attend_dq_kernel<T, DP, RT, kBias>;
    const hipError_t e = allow_lds(kernel, lds);
    if (e != hipSuccess) return e;
    kernel<<<static_cast<unsigned>(xcd_grid(items)), kWave, lds, stream>>>(a, g, tiles, items);
    return hipGetLastError();
}

template <typename T, int DP, bool kBias>
hipError_t launch_dkv(const AttendArgs& a, const AttendGrads& g, hipStream_t stream) {
    const int tiles = (a.k_block + 31) / 32;
    const int64_t items = static_cast<int64_t>(a.blocks) * tiles * a.kv_heads;
    const size_t lds = 2 * kStep * (DP + 16 / sizeof(T)) * sizeof(T) + 6 * kStep * sizeof(float) +
                       (kBias ? static_cast<size_t>(a.share) * a.axes * (2 * a.reach + 1) * sizeof(float) : 0);
    const auto kernel = attend_dkv_kernel<T, DP, kBias>;
    const hipError_t e = allow_lds(kernel, lds);
    if (e != hipSuccess) return e;
    kernel<<<static_cast<unsigned>(xcd_grid(items)), kWave, lds, stream>>>(a, g, tiles, items);
    return hipGetLastError();
}

template <typename T, int DP, bool kBias>
hipError_t launch_pair(const AttendArgs& a, const AttendGrads& g, hipStream_t stream) {
    constexpr int kWide = sizeof(T) == 2 && DP <= 32 ? 4 : 2;
    hipError_t e = a.q_block <= 16 ? launch_dq<T, DP, 1, kBias>(a, g, stream)
                                   : launch_dq<T, DP, kWide, kBias>(a, g, stream);
    if (e != hipSuccess) return e;
    if constexpr (kBias) {
        const int bins = a.axes * a.buckets;
        table_sum_kernel<T><<<bins * a.heads, kWave, 0, stream>>>(g.table_parts, g.parts, a.heads, bins,
                                                                  static_cast<T*>(g.dtable));
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return launch_dkv<T, DP, kBias>(a, g, stream);
}

template <typename T>
hipError_t launch_type(const AttendArgs& a, const AttendGrads& g, hipStream_t stream) {
    const bool bias = a.table != nullptr;
    if (a.D <= 32) return bias ? launch_pair<T, 32, true>(a, g, stream) : launch_pair<T, 32, false>(a, g, stream);
    if (a.D <= 64) return bias ? launch_pair<T, 64, true>(a, g, stream) : launch_pair<T, 64, false>(a, g, stream);
    return bias ? launch_pair<T, 128, true>(a, g, stream) : launch_pair<T, 128, false>(a, g, stream);
}

}  // namespace

int attend_table_parts(int groups, int q_block, int heads) {
    (void)q_block;
    (void)heads;
    return std::max(1, std::min(groups, kTableParts));
}

hipError_t launch_attend_backward(const AttendArgs& a, const AttendGrads& g, bool bf16, hipStream_t stream) {
    return bf16 ? launch_type<__bf16>(a, g, stream) : launch_type<float>(a, g, stream);
}

hipError_t launch_invert(const int32_t* selected, int64_t entries, int blocks, Segment* segs, int64_t tiles,
                         const SortBuffers& sb, int64_t* order, int32_t* runs, hipStream_t stream) {
    int bits = 1;
    while ((int64_t{1} << bits) < int64_t{blocks} + 1) ++bits;
    const SortBits range{0, bits};
    invert_keys_kernel<<<static_cast<unsigned>(tiles), kBlock, 0, stream>>>(
        selected, static_cast<int>(entries), blocks, segs, sb.keys_a, sb.tile_hist, sb.tstride);
    // The buffer that the last pass does not read.
    uint32_t* sorted = range.passes() % 2 == 0 ? sb.keys_a : sb.keys_b;
    hipError_t e = launch_sort(segs, 1, tiles, range, sb, order, sorted, stream);
    if (e != hipSuccess) return e;
    invert_runs_kernel<<<(blocks + 1 + kBlock - 1) / kBlock, kBlock, 0, stream>>>(sorted, static_cast<int>(entries),
                                                                                 blocks, runs);
    return hipGetLastError();
}

}  // namespace tbvh
