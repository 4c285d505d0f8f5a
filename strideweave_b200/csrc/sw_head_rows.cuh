// sw_head_rows.cuh - what surrounds the contractions of the linear head's
// losses (sw_linear_head.cu): the rows that count and their targets, the
// operands' 16-bit planes, the loss from the tiles' statistics, the logits'
// gradient from the kept exponentials, and the gradients' places.
#pragma once

#include "sw_head_gemm.cuh"

namespace sw {
namespace head {

constexpr int kMaxTeacher = SW_MAX_TEACHER;

__device__ __forceinline__ float warp_max(float v) {
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ int warp_sum_int(int v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ bool entry_counts(int index, float logit, int64_t V) {
    return index >= 0 && index < V && logit != -INFINITY;
}

// Estimated microseconds of a contraction in tiles of a shape, the tiles of its
// last, partial wave cut into s parts of the K walk: waves x (stages + what a tile
// hides nowhere), and the traffic of writing and adding the parts.
constexpr int kMaxParts = 64;       // where the tiles do not fill one wave
constexpr int kMaxTailParts = 4;    // of the tiles after whole waves
__host__ __device__ inline int64_t tiles_of(int64_t M, int64_t N, int shape) {
    return ((M + shape_rows(shape) - 1) >> (7 + shape)) * ((N + kBN - 1) / kBN);
}
__host__ __device__ inline float spread_cost(int64_t M, int64_t N, int64_t K, int terms, int shape, int sms, int s) {
    const int workers = shape_workers(shape, sms), steps = int((K + kBK - 1) / kBK);
    const int64_t tiles = tiles_of(M, N, shape);
    const int whole = int(tiles / workers), rest = int(tiles - int64_t(whole) * workers);
    if (s > 1 && (steps < 4 * s || rest == 0 || (whole ? s > kMaxTailParts : rest * s > 2 * workers))) return 1e30f;
    // (a narrow result's tiles compute what they need, but load all of A)
    const float stage = stage_us(shape, terms) * (N <= kBN / 2 ? 0.5f : 1.0f), fixed = fixed_us(shape);
    const float one = float(steps) * stage + fixed, part = float((steps + s - 1) / s) * stage + fixed;
    const float waves = float(whole) * one + float((rest * s + workers - 1) / workers) * part;
    float us = waves;
    if (s > 1) us += 3.0f + float(rest) * float(s) * float(shape_rows(shape) * kBN) * (8.0f / 6.0e6f);
    return us;
}

// Parts that a K walk may be cut into (as above).
__host__ __device__ inline int most_parts(int64_t K) {
    const int64_t s = (K + kBK - 1) / kBK / 4;
    return int(s < 1 ? 1 : s < kMaxParts ? s : kMaxParts);
}
// Rows of fp32 sums that up to `parts` parts of any row count up to M take: all rows,
// and those of the parts past the first, of at most two tiles a worker where the
// tiles do not fill a wave, else of the row groups that the last wave reaches.
__host__ __device__ inline int64_t sum_rows(int64_t M, int64_t N, int parts, int shape, int sms) {
    const int64_t cols = (N + kBN - 1) / kBN, tile_m = shape_rows(shape), all = (M + tile_m - 1) / tile_m * tile_m;
    const int64_t workers = shape_workers(shape, sms), group = 2048 / tile_m;
    const int64_t few = (2 * workers / cols + 1) * tile_m, every = (parts - 1) * all;
    const int64_t reach = (workers / (group * cols) + 2) * group * tile_m;
    const int64_t tail = (reach < all ? reach : all) * ((parts < kMaxTailParts ? parts : kMaxTailParts) - 1);
    const int64_t first = few < every ? few : every;
    return all + (first > tail ? first : tail);
}

constexpr uint32_t kNoMagnitude = 0x7f800000u;  // least magnitude of no rows

// ---- preparation ---------------------------------------------------------------

// flags[t] = 1 when the teacher's row has an entry: a warp per row, one read of
// the teacher (4096 rows of 64 entries 4.4 us, a launch's latency).
__device__ __forceinline__ bool teacher_row_counts(const int* index, const float* logits, int64_t t, int K, int64_t V,
                                                   int lane) {
    bool any = false;
    for (int k = lane; k < K; k += 32) {
        const int i = index[t * K + k];
        if (i >= V) report_device_error(SW_ERR_INVALID);
        any |= entry_counts(i, logits[t * K + k], V);
    }
    return __any_sync(0xffffffffu, any);
}
__global__ void __launch_bounds__(256) teacher_flags_kernel(const int* index, const float* logits, int64_t T, int K,
                                                            int64_t V, uint8_t* flags) {
    pdl_enter();
    const int64_t t = int64_t(blockIdx.x) * 8 + threadIdx.x / 32;
    if (t >= T) return;
    const bool any = teacher_row_counts(index, logits, t, K, V, threadIdx.x & 31);
    if ((threadIdx.x & 31) == 0) flags[t] = any;
}

struct PrepareArgs {
    const int* targets;      // cross entropy, or null
    int ignore_index;
    const int* index;        // distillation
    const float* logits;
    const uint8_t* flags;    // null: every CTA looks at the teacher's rows itself
    int top_k;
    float inv_tau;
    int64_t T, V;
    int rows_pad, entry_tiles;
    const float* upstream;   // null: 1
    int mean;
    float factor;            // c f
    const float* lse;        // a kept lse to start from, or null
    int* row_map;            // compact rows, then the rows that do not count
    uint32_t* row_top;       // to be zeroed for amax_kernel
    int row_tops;
    int* ent_idx;
    float* ent_p;
    float* entropy;
    uint16_t* offs;
    float* coef;             // null: no gradients
    float2* norm;            // what the logits' gradient subtracts, from `lse`
    HeadState* state;
    // the contraction of dh: rows of a launch at most, dim, columns of a piece
    int64_t dh_rows, dh_cols, dh_k;
    int dh_shape, sms, terms;
    // bf16 states, gathered here (null: Float32, split later by split_kernel)
    const uint16_t* h;
    int64_t D, sr, sc;
    int vec;                 // rows are whole aligned 16-byte units
    uint16_t* hc;
    int64_t ld;
};
constexpr int kInlineFlags = 8192;  // teacher entries up to which every CTA looks at all of them

// One teacher row, by a warp: its probabilities and its entries in ascending
// column order, the sum of p log p, and the first entry of every kEntryTile
// columns.
__device__ __forceinline__ void sort_teacher_row(const PrepareArgs& a, int64_t t, int i, int lane, int* cols,
                                                 int* sorted) {
    const int K = a.top_k;
    float top = -INFINITY;
    int n = 0;
    for (int k = lane; k < K; k += 32) {
        const int col = a.index[t * K + k];
        const float x = a.logits[t * K + k];
        const bool ok = entry_counts(col, x, a.V);
        cols[k] = ok ? col : INT_MAX;
        if (ok) {
            top = fmaxf(top, x * a.inv_tau);
            ++n;
        }
    }
    top = warp_max(top);
    n = warp_sum_int(n);
    __syncwarp();
    float sum = 0.0f;
    for (int k = lane; k < K; k += 32)
        if (cols[k] != INT_MAX) sum += expf(a.logits[t * K + k] * a.inv_tau - top);
    sum = warp_sum(sum);
    const float log_sum = logf(sum);
    float ent = 0.0f;
    for (int k = lane; k < K; k += 32) {
        const int col = cols[k];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < K; ++j) rank += (cols[j] < col) || (cols[j] == col && j < k);
        float p = 0.0f;
        if (col != INT_MAX) {
            const float x = a.logits[t * K + k] * a.inv_tau - top;
            p = expf(x) / sum;
            if (p > 0.0f || p != p) ent += p * (x - log_sum);
        }
        sorted[rank] = col;
        a.ent_idx[int64_t(i) * K + rank] = col;
        a.ent_p[int64_t(i) * K + rank] = p;
    }
    ent = warp_sum(ent);
    if (lane == 0) a.entropy[i] = ent;
    __syncwarp();
    for (int tile = lane; tile <= a.entry_tiles; tile += 32) {
        const int64_t col0 = int64_t(tile) * kEntryTile;
        int lo = 0, hi = n;  // entries [0, n) are the real ones
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sorted[mid] < col0) lo = mid + 1;
            else hi = mid;
        }
        a.offs[int64_t(tile) * a.rows_pad + i] = uint16_t(lo);
    }
}

// kRows rows per CTA, and where rows are few a share of their columns.  Each CTA
// counts the rows before its own and all rows that count (T flags from L2: with
// 8 rows a CTA 33 MB in all at T = 8192), so nothing waits for anything:
// row_map[0, count) are the rows that count, in order, row_map[count, T) the
// others.  It then leaves what its rows need: the target entries, the factor of
// their gradient, and in bf16 the states themselves, gathered; the places of
// rows that do not count are zeros.  Bound by the states' way through (4096 x
// 4096: 17.5 us, 3.8 TB/s read and written), else by latency (64 rows of 32
// teacher entries 16 us, most of it the ranks, K comparisons for each entry).
template <int kRows>
__global__ void __launch_bounds__(256) prepare_kernel(const PrepareArgs a) {
    constexpr int kCols = 256;
    __shared__ uint8_t s_flags[kInlineFlags];
    __shared__ int s_before[8], s_total[8], s_bad[8];
    __shared__ int s_dest[kRows];     // compact row, or the place of a row that does not count
    __shared__ uint8_t s_keep[kRows];
    __shared__ __align__(16) int s_sort[8][2 * kMaxTeacher];
    __shared__ __align__(16) uint16_t s_tile[kRows][kCols + 8];
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t t0 = int64_t(blockIdx.x) * kRows;
    const bool inline_flags = !a.targets && !a.flags;
    if (inline_flags) {
        for (int t = tid; t < int(a.T); t += 256) s_flags[t] = 0;
        __syncthreads();
#pragma unroll 4
        for (int e = tid; e < int(a.T) * a.top_k; e += 256) {
            const int i = a.index[e];
            if (i >= a.V) report_device_error(SW_ERR_INVALID);
            if (entry_counts(i, a.logits[e], a.V)) s_flags[e / a.top_k] = 1;
        }
        __syncthreads();
    }
    int before = 0, total = 0, bad = 0;
    auto counts = [&](int64_t t) {
        if (!a.targets) return inline_flags ? s_flags[t] != 0 : a.flags[t] != 0;
        const int y = a.targets[t];
        if (y == a.ignore_index) return false;
        const bool ok = y >= 0 && y < a.V;
        if (!ok) bad = 1;
        return ok;
    };
#pragma unroll 4
    for (int64_t t = tid; t < a.T; t += 256) {
        const int k = counts(t);
        total += k;
        if (t < t0) before += k;
    }
    before = warp_sum_int(before);
    total = warp_sum_int(total);
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
        s_before[warp] = before;
        s_total[warp] = total;
        s_bad[warp] = bad;
    }
    __syncthreads();
    before = total = bad = 0;
    for (int w = 0; w < 8; ++w) {
        before += s_before[w];
        total += s_total[w];
        bad |= s_bad[w];
    }
    if (warp == 0) {
        const int64_t t = t0 + lane;
        const bool mine = lane < kRows && t < a.T;
        const bool keep = mine && counts(t);
        const uint32_t votes = __ballot_sync(0xffffffffu, keep);
        const int rank = before + __popc(votes & ((1u << lane) - 1));
        if (lane < kRows) {
            const int64_t dest = keep ? rank : mine ? a.T - 1 - (t - rank) : t;
            s_dest[lane] = dest < a.rows_pad ? int(dest) : -1;
            s_keep[lane] = keep;
            if (mine && blockIdx.y == 0) a.row_map[dest] = int(t);
            if (keep && blockIdx.y == 0) {
                if (a.targets) a.ent_idx[rank] = a.targets[t];
                if (a.coef) a.coef[rank] = a.mean || !a.upstream ? 1.0f : a.upstream[t];
                if (a.lse) a.norm[rank] = make_float2(a.lse[t], 0.0f);
            }
        }
    }
    __syncthreads();
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) {  // (its rows are mostly padding)
        for (int i = tid; i < a.row_tops; i += 256) a.row_top[i] = 0;
        uint32_t top = 0, least = kNoMagnitude;  // of the row factors (Float32 only)
        if (a.coef && !a.h) {
            for (int64_t t = tid; t < a.T; t += 256)
                if (counts(t)) {
                    const float g = a.mean || !a.upstream ? 1.0f : a.upstream[t];
                    if (isfinite(g)) top = max(top, __float_as_uint(fabsf(g)));
                    if (isfinite(g) && g != 0.0f) least = min(least, __float_as_uint(fabsf(g)));
                }
            top = __reduce_max_sync(0xffffffffu, top);
            least = __reduce_min_sync(0xffffffffu, least);
            if (lane == 0) {
                s_total[warp] = int(top);
                s_before[warp] = int(least);
            }
        }
        __syncthreads();
        if (warp == 0) {
            // the K walk's parts for dh, over the rows that turned out to count:
            // the fewest whose estimate is within 3% of the least
            int splits = 1;
            if (a.dh_cols) {
                const int64_t rows = min(int64_t(total), a.dh_rows);
                const float c0 = spread_cost(rows, a.dh_cols, a.dh_k, a.terms, a.dh_shape, a.sms, lane + 1);
                const float c1 = spread_cost(rows, a.dh_cols, a.dh_k, a.terms, a.dh_shape, a.sms, lane + 33);
                const float least = -warp_max(-fminf(c0, c1)) * 1.03f;
                const uint32_t first = __ballot_sync(0xffffffffu, c0 <= least);
                splits = first ? __ffs(first) : 32 + __ffs(__ballot_sync(0xffffffffu, c1 <= least));
            }
            if (lane == 0) {
                if (a.coef && !a.h)
                    for (int w = 0; w < 8; ++w) {
                        top = max(top, uint32_t(s_total[w]));
                        least = min(least, uint32_t(s_before[w]));
                    }
                HeadState s;
                s.count = total;
                s.bad = bad;
                s.amax[0] = s.amax[1] = 0;
                s.amax[2] = top;
                s.least[0] = s.least[1] = kNoMagnitude;
                s.least[2] = least;
                s.wide = 0;
                // what every row's gradient is multiplied by stays out of the
                // 16-bit logits' gradient: a target's -1 is exact there, where
                // the common factor would round it the same way in every row
                s.grad_scale =
                    a.factor * (a.mean ? (a.upstream && a.coef ? a.upstream[0] : 1.0f) / float(max(total, 1)) : 1.0f);
                s.dh_splits = splits;
                s.done = 0;
                *a.state = s;
                if (bad) report_device_error(SW_ERR_INVALID);
            }
        }
    }
    if (!a.targets && blockIdx.y == 0)
        for (int r = warp; r < kRows; r += 8)
            if (s_keep[r]) sort_teacher_row(a, t0 + r, s_dest[r], lane, s_sort[warp], s_sort[warp] + kMaxTeacher);
    if (!a.h) return;
    // states: row r of this CTA to s_dest[r], and where few rows count again to
    // the places that go with their gradients' remainders
    const bool few = total <= kFewRows && total > 0;
    auto put = [&](int r, int64_t c, const uint4& v) {
        const int d = s_dest[r];
        if (d < 0) return;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        if (s_keep[r]) {
            *reinterpret_cast<uint4*>(a.hc + d * a.ld + c) = v;
            if (few) *reinterpret_cast<uint4*>(a.hc + (d + kFewRows) * a.ld + c) = v;
        } else if (!few || d < kFewRows || d >= kFewRows + total) {
            *reinterpret_cast<uint4*>(a.hc + d * a.ld + c) = zero;
        }
    };
    if (a.vec) {
        const int units = int(a.ld / 8);
        for (int u = blockIdx.y * 256 + tid; u < kRows * units; u += gridDim.y * 256) {
            const int r = u / units, c = (u - r * units) * 8;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (s_keep[r]) v = *reinterpret_cast<const uint4*>(a.h + (t0 + r) * a.sr + c);
            put(r, c, v);
        }
        return;
    }
    const bool by_rows = a.sr == 1 && a.sc != 1;  // walk the unit stride fastest
    for (int64_t c0 = int64_t(blockIdx.y) * kCols; c0 < a.ld; c0 += int64_t(gridDim.y) * kCols) {
        for (int u = tid; u < kRows * kCols; u += 256) {
            const int r = by_rows ? u % kRows : u / kCols, c = by_rows ? u / kRows : u % kCols;
            s_tile[r][c] = s_keep[r] && c0 + c < a.D ? a.h[(t0 + r) * a.sr + (c0 + c) * a.sc] : uint16_t(0);
        }
        __syncthreads();
        for (int u = tid; u < kRows * (kCols / 8); u += 256) {
            const int r = u / (kCols / 8), c = u % (kCols / 8) * 8;
            if (c0 + c < a.ld) put(r, c0 + c, *reinterpret_cast<const uint4*>(&s_tile[r][c]));
        }
        __syncthreads();
    }
}

// ---- 16-bit planes of Float32 operands, and of bf16 weights TMA cannot read ------

struct SplitJob {
    const void* src;
    int64_t rows, cols, sr, sc;
    int vec;                 // rows are whole aligned 16-byte units (Float32: pairs of them)
    const int* row_map;      // null: all rows; else the compact ones, as many as count
    int scale_of;            // index of its magnitude in HeadState::amax
    uint16_t* dst;
    int64_t ld, rows_pad;
    // amax_kernel, contiguous columns: parts of a row, and where there is more than one
    // the rows' magnitudes and how many parts of 32 rows are in them
    int parts;
    uint32_t *row_top, *parts_in;
    unsigned ctas;           // the first CTAs of the grid belong to the first job
};

// Largest finite magnitudes of one or two matrices, for the power of two that
// brings them into f16's range, and of their rows, for whether that will do: a
// warp per row, or where columns are contiguous a CTA per 32 rows, or per part of
// them where rows are few.  Bound by one read (32000 x 2048 Float32 with 900 states
// 51 us, 5.3 TB/s; rows that are not whole vectors, 60000 x 1001, 67 us with eight
// reads a lane in flight, 86 with four).
__global__ void __launch_bounds__(256, 5) amax_kernel(const SplitJob j0, const SplitJob j1, HeadState* state) {
    __shared__ uint32_t s_top[8], s_least[8], s_row[8][32];
    pdl_enter();
    const bool second = blockIdx.x >= j0.ctas;
    const SplitJob& j = second ? j1 : j0;
    const float* x = static_cast<const float*>(j.src);
    const int64_t rows = j.row_map ? state->count : j.rows;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t cta = blockIdx.x - (second ? j0.ctas : 0);
    uint32_t top = 0, least = kNoMagnitude, row = 0;
    auto take = [](uint32_t& row, float v) {
        v = fabsf(v);
        if (v <= 3.402823466e38f) row = max(row, __float_as_uint(v));
    };
    auto row_done = [&](uint32_t m) {
        top = max(top, m);
        if (m) least = min(least, m);
    };
    if (j.sr == 1 && j.sc != 1) {  // read along the unit stride: a lane a row
        const int64_t per = (j.cols + j.parts - 1) / j.parts, items = (rows + 31) / 32 * j.parts;
        for (int64_t t = cta; t < items; t += j.ctas) {
            const int64_t r = t / j.parts * 32 + lane, c0 = t % j.parts * per, c1 = min(c0 + per, j.cols);
            row = 0;
            if (r < rows) {
                const float* p = x + (j.row_map ? int64_t(j.row_map[r]) : r);
                for (int64_t c = c0 + warp; c < c1; c += 64) {
                    float v[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) v[u] = c + 8 * u < c1 ? p[(c + 8 * u) * j.sc] : 0.0f;
#pragma unroll
                    for (int u = 0; u < 8; ++u) take(row, v[u]);
                }
            }
            s_row[warp][lane] = row;
            __syncthreads();
            if (warp == 0) {
                for (int w = 1; w < 8; ++w) row = max(row, s_row[w][lane]);
                bool last = true;
                if (j.parts > 1) {
                    if (row) atomicMax(&j.row_top[r], row);
                    __threadfence();
                    __syncwarp();
                    uint32_t before = 0;
                    if (lane == 0) before = atomicAdd(&j.parts_in[t / j.parts], 1u);
                    last = __shfl_sync(0xffffffffu, before, 0) == uint32_t(j.parts - 1);
                    __threadfence();
                    if (last && r < rows) row = __ldcg(j.row_top + r);
                }
                if (last) row_done(row);
            }
            __syncthreads();
        }
    } else {
        const int64_t step = int64_t(j.ctas) * 8;
        auto start = [&](int64_t o) { return x + (j.row_map ? int64_t(j.row_map[o]) : o) * j.sr; };
        for (int64_t o = cta * 8 + warp; o < rows; o += 2 * step) {
            const float* p = start(o);
            row = 0;
            if (j.vec) {  // two rows at a time, so that one's reads cover the other's reduction
                const bool two = o + step < rows;
                const float* p2 = two ? start(o + step) : p;
                uint32_t row2 = 0;
#pragma unroll 4
                for (int64_t i = lane * 4; i < j.cols; i += 128) {
                    const float4 v = *reinterpret_cast<const float4*>(p + i);
                    const float4 v2 = *reinterpret_cast<const float4*>(p2 + i);
                    take(row, v.x);
                    take(row, v.y);
                    take(row, v.z);
                    take(row, v.w);
                    take(row2, v2.x);
                    take(row2, v2.y);
                    take(row2, v2.z);
                    take(row2, v2.w);
                }
                row_done(__reduce_max_sync(0xffffffffu, row));
                row_done(__reduce_max_sync(0xffffffffu, row2));
                continue;
            }
            for (int64_t q = o; q < rows && q <= o + step; q += step) {
                p = start(q);
                row = 0;
                for (int64_t i = lane; i < j.cols; i += 256) {
                    float v[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) v[u] = i + 32 * u < j.cols ? p[(i + 32 * u) * j.sc] : 0.0f;
#pragma unroll
                    for (int u = 0; u < 8; ++u) take(row, v[u]);
                }
                row_done(__reduce_max_sync(0xffffffffu, row));
            }
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    least = __reduce_min_sync(0xffffffffu, least);
    if (lane == 0) {
        s_top[warp] = top;
        s_least[warp] = least;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 8; ++w) {
            top = max(top, s_top[w]);
            least = min(least, s_least[w]);
        }
        if (top) atomicMax(&state->amax[j.scale_of], top);
        atomicMin(&state->least[j.scale_of], least);
    }
}

// One or two matrices into operands [rows_pad][ld]: a copy of bf16 values, or
// two f16 planes of a Float32 value times 2^q (hi rounded to nearest, lo the
// rest), or three bf16 ones.  Rows past the ones that count are zero.  Bound by a read and a write of
// the matrix (32000 x 1024 Float32 with its 2048 states 57 us, 4.9 TB/s; bf16
// 60000 x 1001, which TMA cannot read, 56 us, 4.3 TB/s).  Rows that are not whole
// vectors are read element by element: aligned vectors shifted into place took
// the same time.
template <bool kF32>
__global__ void __launch_bounds__(256) split_kernel(const SplitJob j0, const SplitJob j1, HeadState* state) {
    __shared__ float tile[32][33];
    pdl_enter();
    const bool second = blockIdx.x >= j0.ctas;
    const SplitJob& j = second ? j1 : j0;
    const int64_t cta = blockIdx.x - (second ? j0.ctas : 0);
    const int64_t valid = j.row_map ? min(j.rows, int64_t(state->count)) : j.rows;
    const bool wide = kF32 && rows_far_apart(state);
    if (kF32 && blockIdx.x == 0 && threadIdx.x == 0) state->wide = wide;
    const float scale = kF32 ? pow2i(scale_exponent(state->amax[j.scale_of], wide)) : 1.0f;
    if (j.sc == 1) {
        // a thread writes 8 columns; it reads them as vectors where rows are
        // aligned, else one by one (neighbouring threads share the sectors)
        const int64_t units = j.ld / 8;
#pragma unroll 2
        for (int64_t u = cta * 256 + threadIdx.x; u < j.rows_pad * units; u += int64_t(j.ctas) * 256) {
            const int64_t r = u / units, c = (u - r * units) * 8;
            uint4 hi = make_uint4(0, 0, 0, 0), lo = hi, third = hi;
            if (r < valid) {
                const int64_t at = (j.row_map ? int64_t(j.row_map[r]) : r) * j.sr + c;
                if (kF32) {
                    const float* p = static_cast<const float*>(j.src) + at;
                    float v[8];
                    if (j.vec) {
                        const float4 *q = reinterpret_cast<const float4*>(p), a = q[0], b = q[1];
                        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
                    } else {
#pragma unroll
                        for (int q = 0; q < 8; ++q) v[q] = c + q < j.cols ? p[q] : 0.0f;
                    }
                    auto plane = [&]() {
                        uint32_t h[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) h[q] = split2(wide, v[2 * q], v[2 * q + 1]);
                        return make_uint4(h[0], h[1], h[2], h[3]);
                    };
#pragma unroll
                    for (int q = 0; q < 8; ++q) v[q] *= scale;
                    hi = plane();
                    lo = plane();
                    if (wide) third = plane();
                } else {
                    const uint16_t* p = static_cast<const uint16_t*>(j.src) + at;
                    if (j.vec) {
                        hi = *reinterpret_cast<const uint4*>(p);
                    } else {
                        uint32_t w[8];
#pragma unroll
                        for (int q = 0; q < 8; ++q) w[q] = c + q < j.cols ? p[q] : 0;
                        hi = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
                    }
                }
            }
            *reinterpret_cast<uint4*>(j.dst + r * j.ld + c) = hi;
            if (kF32) *reinterpret_cast<uint4*>(j.dst + (j.rows_pad + r) * j.ld + c) = lo;
            if (wide) *reinterpret_cast<uint4*>(j.dst + (2 * j.rows_pad + r) * j.ld + c) = third;
        }
        return;
    }
    // 32 x 32 tiles through shared memory, read along the unit stride
    const bool by_rows = j.sr == 1;
    const int x = threadIdx.x & 31, y0 = threadIdx.x >> 5;
    const int64_t tiles_c = (j.ld + 31) / 32, tiles = (j.rows_pad + 31) / 32 * tiles_c;
    for (int64_t t = cta; t < tiles; t += j.ctas) {
        const int64_t r0 = t / tiles_c * 32, c0 = t % tiles_c * 32;
        for (int y = y0; y < 32; y += 8) {
            const int64_t r = r0 + (by_rows ? x : y), c = c0 + (by_rows ? y : x);
            float v = 0.0f;
            if (r < valid && c < j.cols) {
                const int64_t at = (j.row_map ? int64_t(j.row_map[r]) : r) * j.sr + c * j.sc;
                v = kF32 ? static_cast<const float*>(j.src)[at]
                         : __bfloat162float(static_cast<const __nv_bfloat16*>(j.src)[at]);
            }
            tile[by_rows ? x : y][by_rows ? y : x] = v;
        }
        __syncthreads();
        for (int y = y0; y < 32; y += 8) {
            const int64_t r = r0 + y, c = c0 + x;
            if (r < j.rows_pad && c < j.ld) {
                const float v = tile[y][x];
                if (kF32) {
                    float s = v * scale, none = 0.0f;
                    for (int plane = 0; plane < (wide ? 3 : 2); ++plane)
                        j.dst[(plane * j.rows_pad + r) * j.ld + c] = uint16_t(split2(wide, s, none));
                } else {
                    j.dst[r * j.ld + c] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
                }
            }
        }
        __syncthreads();
    }
}

// ---- after the logits ------------------------------------------------------------

struct LossArgs {
    const float4* partial;   // [rows][slots]
    int slots, slot_shift;
    int row0, rows;          // compact rows [row0, row0 + rows), a CTA each
    int all_rows;            // CTAs over all launches that write a row's loss
    HeadState* state;
    const int* row_map;
    const int* targets;
    int ignore_index;
    const float* entropy;    // distillation, or null
    float factor;            // f
    float logit_scale;
    float* row_loss;         // compact
    float2* norm;            // compact: for gradients that start from the logits again
    float* loss;             // per row, or the mean; null: neither
    int mean;
    float* lse;              // per row, or null
    // the logits' gradient from the kept exponentials (grad null: none)
    uint16_t* grad;          // of row row0
    int64_t ld_grad, V, seg; // seg: columns of a CTA
    const float* coef;       // compact, as the entries
    const int* ent_idx;
    const float* ent_p;
    const float* ent_s;
    int ent_k;
};

// A row's statistics from its half tiles', its loss, and (grad) the gradient of
// its logits: exp2(k2 (z - top)) of a half tile times exp2(k2 (top - ref)) / sum
// is the softmax, in place of the stored exponentials, and the target entries
// are written from their own Float32 z (where the softmax is near p, the stored
// 11 bits of it would not be enough).  A row's largest z and the logarithm of
// its sum stay apart until the end: added up, their rounding is all that a row
// sure of its target would have left.  A thread takes 8 columns (bf16), a warp a block of 64
// (Float32: hi and lo values replace the block they were computed from).  The
// last row to be done adds up the mean, in a fixed order.  Bound by the
// exponentials' read and write, part of them still in L2: 4096 x 32000 110 us, 4.8
// TB/s (Float32 2048 x 32000 116).  One reference for a whole row instead of one a
// half tile would spare this pass, at the cost of one more 16-bit rounding, of
// the states in dw, and of a target's exact -1: not taken.
template <bool kF32>
__global__ void __launch_bounds__(256, kF32 ? 4 : 3) loss_kernel(const LossArgs a) {
    constexpr int kSub = kF32 ? 2048 : 8192;  // columns of a batch: four loads a thread
    __shared__ float factor[kSub / 64];
    __shared__ float4 s_stat[8];
    __shared__ float s_part[8];
    __shared__ int s_last;
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // the last rows first: they are the ones the contraction left in L2, and the
    // next one starts with the first
    const int64_t i = int64_t(gridDim.x) - 1 - blockIdx.x;
    const bool writes = blockIdx.y == 0;
    const int count = a.state->rows(a.row0);
    const float k2 = a.logit_scale * kLog2e;
    float ref = -INFINITY, log2_sum = 0.0f;
    // the first 8192 columns' exponentials are on their way while the statistics
    // are added up, and later each batch while the one before it is written
    const int64_t c_begin = int64_t(blockIdx.y) * a.seg, c_end = min(c_begin + a.seg, a.V);
    uint16_t* row = a.grad + i * a.ld_grad;
    uint4 held[4];
    auto fetch = [&](int64_t c0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t c = c0 + (kF32 ? 64 * warp + 512 * j : tid * 8 + 2048 * j);
            if (c >= c_end) continue;
            if (kF32) {
                const float2 v = reinterpret_cast<const float2*>(row + 2 * c)[lane];
                held[j].x = __float_as_uint(v.x);
                held[j].y = __float_as_uint(v.y);
            } else {
                held[j] = *reinterpret_cast<const uint4*>(row + c);
            }
        }
    };
    if (a.grad && i < count) fetch(c_begin);
    if (i < count) {
        const float4* part = a.partial + i * a.slots;
        // against the largest z of a thread's slots, of a warp's, and then of all
        auto finite = [](float r) { return r == -INFINITY ? 0.0f : r; };
        float sum = 0.0f, dot = 0.0f;
#pragma unroll 4
        for (int t = tid; t < a.slots; t += 256) {
            const float4 p = part[t];
            const float next = fmaxf(ref, p.x), base = finite(next);
            sum = sum * ex2((ref - base) * k2) + p.y * ex2((p.x - base) * k2);
            dot += p.z;
            ref = next;
        }
        const float own = ref;
        ref = warp_max(ref);
        sum = warp_sum(sum * ex2((own - finite(ref)) * k2));
        dot = warp_sum(dot);
        if (lane == 0) s_stat[warp] = make_float4(ref, sum, dot, 0.0f);
        __syncthreads();
        for (int w = 0; w < 8; ++w) ref = fmaxf(ref, s_stat[w].x);
        sum = dot = 0.0f;
        for (int w = 0; w < 8; ++w) {
            const float4 p = s_stat[w];
            sum += p.y * ex2((p.x - finite(ref)) * k2);
            dot += p.z;
        }
        log2_sum = log2f(sum);
        if (writes && tid == 0) {
            // (where the target is the largest, ref - dot is 0: a small loss keeps its digits)
            const float v = a.factor * ((a.entropy ? a.entropy[a.row0 + i] : 0.0f) +
                                        (log2_sum * kLn2 + (ref - dot) * a.logit_scale));
            const int64_t row = a.row_map[a.row0 + i];
            a.row_loss[a.row0 + i] = v;
            a.norm[a.row0 + i] = make_float2(ref, log2_sum);
            if (a.loss && !a.mean) a.loss[row] = v;
            if (a.lse) a.lse[row] = fmaf(ref, a.logit_scale, log2_sum * kLn2);
        }
    } else if (writes && tid == 0 && i < a.rows) {
        const int64_t row = a.row_map[a.row0 + i];
        float v = 0.0f;
        if (a.targets && a.targets[row] != a.ignore_index) v = NAN;  // a target outside the vocabulary
        if (a.loss && !a.mean) a.loss[row] = v;
        if (a.lse) a.lse[row] = 0.0f;
    }
    if (writes && a.mean) {
        if (tid == 0) {
            __threadfence();
            s_last = atomicAdd(&a.state->done, 1) == a.all_rows - 1;
        }
        __syncthreads();
        if (s_last) {
            __threadfence();
            float s = 0.0f;
            for (int r = tid; r < a.state->count; r += 256) s += __ldcg(a.row_loss + r);
            s = warp_sum(s);
            __syncthreads();
            if (lane == 0) s_part[warp] = s;
            __syncthreads();
            if (tid == 0) {
                s = 0.0f;
                for (int w = 0; w < 8; ++w) s += s_part[w];
                *a.loss = a.state->bad ? NAN : s / float(a.state->count);
            }
        }
    }
    if (!a.grad || i >= count) return;
    const bool few = !kF32 && a.state->few(a.row0), wide = kF32 && a.state->wide;
    const float coef = a.coef[a.row0 + i] * (kF32 ? pow2i(scale_exponent(a.state->amax[2], wide)) : 1.0f);
    uint16_t* rest = row + kFewRows * a.ld_grad;
    for (int64_t c0 = c_begin; c0 < c_end; c0 += kSub) {
        const int64_t c1 = min(c0 + kSub, c_end);
        __syncthreads();
        for (int t = tid; t < int((c1 - c0 + 63) / 64); t += 256) {
            const float top = a.partial[i * a.slots + ((c0 + t * 64) >> a.slot_shift)].x;
            // (a half tile of nothing but -inf stored zeros)
            factor[t] = top == -INFINITY
                            ? 0.0f
                            : ex2((top - ref) * k2 - log2_sum) * coef * (kF32 ? 1.0f : 1.0f / 32768.0f);
        }
        __syncthreads();
        uint4 now[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) now[j] = held[j];
        if (c1 < c_end) fetch(c1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t c = c0 + (kF32 ? 64 * warp + 512 * j : tid * 8 + 2048 * j);
            if (c >= c1) continue;
            const float f = factor[(c - c0) / 64];
            if (kF32) {
                float2 v = make_float2(__uint_as_float(now[j].x), __uint_as_float(now[j].y));
                v.x = c + 2 * lane < a.V ? v.x * f : 0.0f;
                v.y = c + 2 * lane + 1 < a.V ? v.y * f : 0.0f;
                const uint32_t hi = split2(wide, v.x, v.y), lo = split2(wide, v.x, v.y);
                __syncwarp();  // (the whole block was read before any of it is replaced)
                reinterpret_cast<uint32_t*>(row + 2 * c)[lane] = hi;
                reinterpret_cast<uint32_t*>(row + 2 * c + 64)[lane] = lo;
            } else {
                const uint32_t e[4] = {now[j].x, now[j].y, now[j].z, now[j].w};
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float2 g = __half22float2(*reinterpret_cast<const __half2*>(&e[q]));
                    g.x *= f;
                    g.y *= f;
                    const __nv_bfloat162 h = __floats2bfloat162_rn(g.x, g.y);
                    hi[q] = *reinterpret_cast<const uint32_t*>(&h);
                    lo[q] = pack2<true>(g.x - __low2float(h), g.y - __high2float(h));
                }
                *reinterpret_cast<uint4*>(row + c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if (few) *reinterpret_cast<uint4*>(rest + c) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
    }
    __syncthreads();  // the entries overwrite what the loop above wrote
    for (int k = tid; k < a.ent_k; k += 256) {
        const int64_t at = (a.row0 + i) * a.ent_k + k;
        const int col = a.ent_idx[at];
        if (col < c_begin || col >= c_end || (k > 0 && a.ent_idx[at - 1] == col)) continue;
        float p = a.ent_p ? a.ent_p[at] : 1.0f;
        for (int j = 1; k + j < a.ent_k && a.ent_idx[at + j] == col; ++j) p += a.ent_p[at + j];
        float g = (ex2((a.ent_s[at] - ref) * k2 - log2_sum) - p) * coef;
        if (kF32) {
            uint16_t* d = row + (col & ~63) * int64_t(2) + (col & 63);
            float none = 0.0f;
            d[0] = uint16_t(split2(wide, g, none));
            d[64] = uint16_t(split2(wide, g, none));
        } else {
            const __nv_bfloat16 hi = __float2bfloat16_rn(g);
            row[col] = __bfloat16_as_ushort(hi);
            if (few) rest[col] = __bfloat16_as_ushort(__float2bfloat16_rn(g - __bfloat162float(hi)));
        }
    }
}

// ---- after the gradients' contractions ---------------------------------------------

// Result rows from the fp32 sums of the K walk's parts, added in order (so the
// same call gives the same bits), to their places; with by_count, zeros in the
// rows that do not count.  Bound by the sums' read, mostly from L2.
struct PlaceArgs {
    const float* sums;       // rows as Walk places them
    int64_t ld;
    int splits, tile_m, workers;  // splits 0: state->dh_splits
    int64_t rows, cols;
    const HeadState* state;
    int by_count, row0;
    const int* row_map;
    void* dst;
    int64_t dst_row, dst_col;
    int vec;                 // dst rows are contiguous and aligned to four elements
};
template <bool kF32, int kRows>
__global__ void __launch_bounds__(256) place_kernel(const PlaceArgs a) {
    pdl_enter();
    const int splits = a.splits > 0 ? a.splits : a.state->dh_splits;
    const int64_t summed = a.by_count ? min(a.rows, int64_t(a.state->rows(a.row0))) : a.rows;
    const bool few = !kF32 && a.by_count && a.state->few(a.row0);  // their remainders are further rows
    const Walk walk(few ? kFewRows + int(summed) : int(summed), int((a.cols + kBN - 1) / kBN), a.tile_m, a.workers,
                    splits);
    // a CTA takes 1024 columns of kRows rows (of one tile) at a time: with four,
    // a thread has four reads in flight where one left it waiting (4096 x 4096:
    // 60 us with one row, 33 so); with few rows and many parts to add, CTAs are
    // worth more (64 x 2048: 10 us with one row, 17 with four)
    const int64_t c = int64_t(blockIdx.x) * 1024 + threadIdx.x * 4;
    if (c >= a.cols) return;
    for (int64_t m0 = int64_t(blockIdx.y) * kRows; m0 < a.rows; m0 += int64_t(gridDim.y) * kRows) {
        float4 s[kRows];
#pragma unroll
        for (int j = 0; j < kRows; ++j) s[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (m0 < summed) {
            const int parts = walk.tile_of(int(m0) / a.tile_m, int(c) / kBN) < walk.whole ? 1 : splits;
            for (int rest = 0; rest <= (few ? kFewRows : 0); rest += kFewRows) {
#pragma unroll(8 / kRows)
                for (int k = 0; k < parts; ++k) {
                    // (ld is whole groups of four)
                    const float* p = a.sums + int64_t(walk.sum_row(k, int(m0) + rest)) * a.ld + c;
#pragma unroll
                    for (int j = 0; j < kRows; ++j)
                        if (m0 + j < summed) {
                            const float4 v = *reinterpret_cast<const float4*>(p + j * a.ld);
                            s[j].x += v.x;
                            s[j].y += v.y;
                            s[j].z += v.z;
                            s[j].w += v.w;
                        }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const int64_t m = m0 + j;
            if (m >= a.rows) break;
            const int64_t at = (a.row_map ? int64_t(a.row_map[m]) : m) * a.dst_row + c * a.dst_col;
            if (a.vec && c + 4 <= a.cols) {
                if (kF32) *reinterpret_cast<float4*>(static_cast<float*>(a.dst) + at) = s[j];
                else
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.dst) + at) =
                        make_uint2(pack2<true>(s[j].x, s[j].y), pack2<true>(s[j].z, s[j].w));
                continue;
            }
            const float r[4] = {s[j].x, s[j].y, s[j].z, s[j].w};
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c + q < a.cols) {
                    if (kF32) static_cast<float*>(a.dst)[at + q * a.dst_col] = r[q];
                    else static_cast<__nv_bfloat16*>(a.dst)[at + q * a.dst_col] = __float2bfloat16_rn(r[q]);
                }
        }
    }
}

// A result that TMA could not write where it belongs, from rows padded to whole
// 16 bytes: dense destinations as aligned 16-byte vectors whatever their rows'
// alignment (reads of neighbouring threads share sectors), others element by
// element.  Bound by a read and a write (60000 x 1001 in bf16 57 us, 4.2 TB/s, in
// Float32 101 us, 4.8 TB/s).
template <class E>
__global__ void __launch_bounds__(256) unpad_kernel(const E* src, int64_t ld, int64_t rows, int64_t cols, E* dst,
                                                    int64_t dst_row, int64_t dst_col) {
    pdl_enter();
    constexpr int kPer = 16 / sizeof(E);
    const int64_t n = rows * cols, step = int64_t(gridDim.x) * 256, first = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (dst_col == 1 && (dst_row == cols || rows == 1)) {
        const int64_t head = min(n, int64_t((16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15) / int64_t(sizeof(E)));
        const int64_t vectors = (n - head) / kPer;
        for (int64_t v = first; v < vectors; v += step) {
            const int64_t f = head + v * kPer;
            int64_t r = f / cols, c = f - r * cols;
            __align__(16) E e[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                e[j] = src[r * ld + c];
                if (++c == cols) {
                    c = 0;
                    ++r;
                }
            }
            *reinterpret_cast<uint4*>(dst + f) = *reinterpret_cast<const uint4*>(e);
        }
        const int64_t tail = head + vectors * kPer;
        for (int64_t f = first; f < n - (tail - head); f += step) {
            const int64_t g = f < head ? f : tail + (f - head), r = g / cols;
            dst[g] = src[r * ld + (g - r * cols)];
        }
        return;
    }
    const bool by_rows = dst_row == 1 && dst_col != 1;  // walk the unit stride fastest
    const int64_t inner = by_rows ? rows : cols;
    for (int64_t f = first; f < n; f += step) {
        const int64_t o = f / inner, i = f - o * inner, r = by_rows ? i : o, c = by_rows ? o : i;
        dst[r * dst_row + c * dst_col] = src[r * ld + c];
    }
}

}  // namespace head
}  // namespace sw
