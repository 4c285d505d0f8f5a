// sw_linear_head.cu - losses of a linear head over a large vocabulary, with
// their gradients and without keeping the logits.
//
//   s[t, v] = c sum_d h[t, d] w[v, d]       lse_t = log sum_v exp(s[t, v])
//   cross entropy  loss_t = lse_t - s[t, y_t]
//   distillation   loss_t = tau^2 (sum_k p_tk (log p_tk - s[t, i_tk]) + lse_t),   c = 1 / tau,
//                  p_t = softmax of the teacher's entries / tau
//   dlogits  G[t, v] = g_t c f (exp(s[t, v] - lse_t) - sum_k p_tk [v = i_tk])     (f = 1 or tau^2)
//   dh = G w,  dw = G^T h
//
// Cross entropy is the case of one entry with p = 1, so both run the same
// kernels.  The rows that count are gathered first (a row that is ignored, or
// whose teacher has no entry, costs nothing and its states are never read);
// the contractions of sw_head_gemm.cuh then run over the compact rows.  The
// forward keeps a (max, sum, target term) triple per row and column tile; the
// backward walks the vocabulary in pieces: the piece's logits are computed
// again, their gradient is rounded once to the operand type, and two more
// contractions take it to dh (summed over the pieces in fp32) and dw.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "sw_common.cuh"
#include "sw_head_gemm.cuh"
#include "sw_ptx.cuh"
#include "sw_tma.cuh"

namespace sw {
namespace head {
namespace {

constexpr int kMaxTeacher = SW_MAX_TEACHER;
constexpr int64_t kDefaultWorkspace = int64_t(4) << 30;

__device__ __forceinline__ float warp_max(float v) {
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ bool entry_counts(int index, float logit, int64_t V) {
    return index >= 0 && index < V && logit != -INFINITY;
}

// ---- preparation ---------------------------------------------------------------

// flags[t] = 1 when the teacher's row has an entry (a warp per row).
__global__ void teacher_flags_kernel(const int* index, const float* logits, int64_t T, int K, int64_t V,
                                     uint8_t* flags) {
    pdl_enter();
    const int64_t t = int64_t(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
    const int lane = threadIdx.x & 31;
    if (t >= T) return;
    bool any = false;
    for (int k = lane; k < K; k += 32) {
        const int i = index[t * K + k];
        if (i >= V) report_device_error(SW_ERR_INVALID);
        any |= entry_counts(i, logits[t * K + k], V);
    }
    any = __any_sync(0xffffffffu, any);
    if (lane == 0) flags[t] = any;
}

// Estimated microseconds of a contraction in tiles of a shape, the tiles of its
// last, partial wave cut into s parts of the K walk: waves x (stages + a tile's
// cost that nothing hides), and the traffic of writing and adding the parts.  A
// K stage takes 0.27 us (kSingle: 128 x 256 on one SM, kPair2: 256 x 256 on two)
// or 0.52 (kTall), a tile's fill and drain 2 us (kTall: 5), an adding launch 3.
constexpr int kMaxParts = 64;       // where the tiles do not fill one wave
constexpr int kMaxTailParts = 4;    // of the tiles after whole waves
__host__ __device__ inline int shape_workers(int shape, int sms) { return shape == kSingle ? sms : sms / 2; }
__host__ __device__ inline float spread_cost(int64_t M, int64_t N, int64_t K, int terms, int shape, int sms, int s) {
    const int workers = shape_workers(shape, sms), steps = int((K + kBK - 1) / kBK);
    const int64_t tiles = ((M + shape_rows(shape) - 1) >> (7 + shape)) * ((N + kBN - 1) / kBN);
    const int whole = int(tiles / workers), rest = int(tiles - int64_t(whole) * workers);
    if (s > 1 && (steps < 4 * s || rest == 0 || (whole ? s > kMaxTailParts : rest * s > 2 * workers))) return 1e30f;
    const float stage = float(terms) * (shape == kTall ? 0.52f : 0.27f), fixed = shape == kTall ? 5.0f : 2.0f;
    const int share = (steps + s - 1) / s;
    float us = float(whole) * (float(steps) * stage + fixed) +
               float((rest * s + workers - 1) / workers) * (float(share) * stage + fixed);
    if (s > 1) us += 3.0f + float(rest) * float(s) * float(shape_rows(shape) * kBN) * (8.0f / 6.0e6f);
    return us;
}

struct RowsArgs {
    const int* targets;      // cross entropy, or null
    int ignore_index;
    const uint8_t* flags;    // distillation
    int64_t T, V;
    const float* upstream;   // null: 1
    int mean;
    float factor;            // c f
    const float* lse;        // a kept lse to start from, or null
    int* row_map;            // compact rows, then the rows that do not count
    int* ent_idx;            // cross entropy: the compact rows' targets
    float* coef;
    float* lse2;
    HeadState* state;
    int64_t dh_rows, dh_cols, dh_k;  // the contraction of dh: rows of a launch at most, dim, columns of a piece
    int dh_shape, sms, terms;
};

// One CTA ranks the rows, four per thread and pass: row_map[0, count) are the
// rows that count, in order, row_map[count, T) the others.
__global__ void __launch_bounds__(1024) rows_kernel(const RowsArgs a) {
    __shared__ int warp_n[32];
    __shared__ int total;
    __shared__ float cost[kMaxParts];
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int kept = 0, bad = 0;
    uint32_t top = 0;
    for (int64_t base = 0; base < a.T; base += 4096) {
        const int64_t t0 = base + tid * 4;
        int y[4];
        uint32_t keep = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            y[j] = 0;
            if (t0 + j >= a.T) continue;
            if (a.targets) {
                y[j] = a.targets[t0 + j];
                if (y[j] != a.ignore_index) {
                    if (y[j] >= 0 && y[j] < a.V) keep |= 1u << j;
                    else bad = 1;
                }
            } else if (a.flags[t0 + j]) {
                keep |= 1u << j;
            }
        }
        int n = __popc(keep);
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= o) n += up;
        }
        if (lane == 31) warp_n[warp] = n;
        __syncthreads();
        if (warp == 0) {
            int w = warp_n[lane];
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) w += up;
            }
            warp_n[lane] = w;
            if (lane == 31) total = w;
        }
        __syncthreads();
        int before = kept + (warp ? warp_n[warp - 1] : 0) + n - __popc(keep);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t t = t0 + j;
            if (t >= a.T) continue;
            if (keep >> j & 1) {
                a.row_map[before] = int(t);
                if (a.targets) a.ent_idx[before] = y[j];
                if (a.coef) {
                    const float g = a.mean || !a.upstream ? 1.0f : a.upstream[t];
                    a.coef[before] = g;
                    if (isfinite(g)) top = max(top, __float_as_uint(fabsf(g)));
                }
                if (a.lse) a.lse2[before] = a.lse[t] * kLog2e;
                ++before;
            } else {
                a.row_map[a.T - 1 - (t - before)] = int(t);
            }
        }
        kept += total;
        __syncthreads();
    }
    if (a.coef && top) atomicMax(&a.state->amax[2], top);
    // the K walk's parts for dh, over the rows that turned out to count
    if (tid < kMaxParts) {
        const int64_t rows = min(int64_t(kept), a.dh_rows);
        cost[tid] = spread_cost(rows, a.dh_cols, a.dh_k, a.terms, a.dh_shape, a.sms, tid + 1);
    }
    bad = __syncthreads_or(bad);
    if (tid == 0) {
        a.state->count = kept;
        a.state->bad = bad;
        if (bad) report_device_error(SW_ERR_INVALID);
        // what every row's gradient is multiplied by stays out of the 16-bit
        // logits' gradient: a target's -1 is exact there, where the common
        // factor would round it the same way in every row
        a.state->grad_scale =
            a.factor * (a.mean ? (a.upstream ? a.upstream[0] : 1.0f) / float(max(kept, 1)) : 1.0f);
        int best = 0;
        for (int s = 1; s < kMaxParts; ++s)
            if (cost[s] < cost[best] * 0.97f) best = s;
        a.state->dh_splits = best + 1;
    }
}

// A warp per compact row: its teacher's probabilities and its entries in
// ascending column order, the row's sum of p log p, and the first entry of
// every kEntryTile columns.
__global__ void teacher_sort_kernel(const int* index, const float* logits, int K, int64_t V, float inv_tau,
                                    const int* row_map, const HeadState* state, int rows_pad, int tiles,
                                    int* ent_idx, float* ent_p, float* entropy, uint16_t* offs) {
    __shared__ int s_idx[4][kMaxTeacher];
    __shared__ int s_sorted[4][kMaxTeacher];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i = blockIdx.x * 4 + warp;
    if (i >= state->count) return;
    const int64_t t = row_map[i];
    float top = -INFINITY;
    for (int k = lane; k < K; k += 32) {
        const int col = index[t * K + k];
        const float x = logits[t * K + k];
        const bool ok = entry_counts(col, x, V);
        s_idx[warp][k] = ok ? col : INT_MAX;
        if (ok) top = fmaxf(top, x * inv_tau);
    }
    top = warp_max(top);
    __syncwarp();
    float sum = 0.0f;
    for (int k = lane; k < K; k += 32)
        if (s_idx[warp][k] != INT_MAX) sum += expf(logits[t * K + k] * inv_tau - top);
    sum = warp_sum(sum);
    const float log_sum = logf(sum);
    float ent = 0.0f;
    int n = 0;
    for (int k = lane; k < K; k += 32) {
        const int col = s_idx[warp][k];
        int rank = 0;
        for (int j = 0; j < K; ++j) {
            const int o = s_idx[warp][j];
            rank += (o < col) || (o == col && j < k);
        }
        float p = 0.0f;
        if (col != INT_MAX) {
            const float x = logits[t * K + k] * inv_tau - top;
            p = expf(x) / sum;
            if (p > 0.0f || p != p) ent += p * (x - log_sum);
            ++n;
        }
        s_sorted[warp][rank] = col;
        ent_idx[int64_t(i) * K + rank] = col;
        ent_p[int64_t(i) * K + rank] = p;
    }
    ent = warp_sum(ent);
    if (lane == 0) entropy[i] = ent;
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    __syncwarp();
    for (int tile = lane; tile <= tiles; tile += 32) {
        const int64_t col0 = int64_t(tile) * kEntryTile;
        int lo = 0, hi = n;  // entries [0, n) are the real ones
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s_sorted[warp][mid] < col0) lo = mid + 1;
            else hi = mid;
        }
        offs[int64_t(tile) * rows_pad + i] = uint16_t(lo);
    }
}

// Largest finite magnitude of a matrix (of the rows of row_map when it is
// given): a warp per row, or per column where columns are contiguous; `vec`:
// rows are whole aligned groups of four.
__global__ void __launch_bounds__(256) amax_kernel(const float* x, int64_t rows, int64_t cols, int64_t sr, int64_t sc,
                                                   int vec, const int* row_map, const HeadState* count_from,
                                                   uint32_t* out) {
    pdl_enter();
    if (count_from) rows = count_from->count;
    const bool by_rows = sr == 1 && sc != 1;  // walk the unit stride fastest
    const int64_t outer = by_rows ? cols : rows, inner = by_rows ? rows : cols;
    const int64_t so = by_rows ? sc : sr, si = by_rows ? sr : sc;
    const int lane = threadIdx.x & 31;
    const int64_t warps = int64_t(gridDim.x) * 8;
    uint32_t top = 0;
    auto take = [&](float v) {
        v = fabsf(v);
        if (v <= 3.402823466e38f) top = max(top, __float_as_uint(v));
    };
    for (int64_t o = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); o < outer; o += warps) {
        const float* p = x + (by_rows ? o : row_map ? int64_t(row_map[o]) : o) * so;
        if (vec) {
#pragma unroll 4
            for (int64_t i = lane * 4; i < inner; i += 128) {
                const float4 v = *reinterpret_cast<const float4*>(p + i);
                take(v.x);
                take(v.y);
                take(v.z);
                take(v.w);
            }
        } else {
#pragma unroll 4
            for (int64_t i = lane; i < inner; i += 32) take(p[(by_rows && row_map ? int64_t(row_map[i]) : i) * si]);
        }
    }
    for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0 && top) atomicMax(out, top);
}

// pack_kernel for rows that are whole aligned 16-byte units (8 columns at a
// time, coalesced): a gather of bf16 rows, or the split of Float32 rows.
template <bool kF32>
__global__ void __launch_bounds__(256) pack_rows_kernel(const void* src, int64_t rows, int64_t cols, int64_t sr,
                                                        const int* row_map, const HeadState* state, int use_count,
                                                        int scale_of, uint16_t* dst, int64_t ld, int64_t rows_pad) {
    pdl_enter();
    const int64_t valid = use_count ? min(rows, int64_t(state->count)) : rows;
    const bool twice = !kF32 && use_count && state->few(0);  // the rows again for their gradients' remainders
    const float scale = kF32 ? pow2i(scale_exponent(state->amax[scale_of])) : 1.0f;
    const int64_t units = cols / 8;  // ld == cols here
    const int64_t stride = int64_t(gridDim.x) * 256;
#pragma unroll 2
    for (int64_t u = int64_t(blockIdx.x) * 256 + threadIdx.x; u < rows_pad * units; u += stride) {
        const int64_t r = u / units, c = (u - r * units) * 8;
        const int64_t from = twice && r >= kFewRows ? r - kFewRows : r;
        uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
        if (from < valid) {
            const int64_t at = (row_map ? int64_t(row_map[from]) : from) * sr + c;
            if (kF32) {
                const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(src) + at);
                const float4 a = p[0], b = p[1];
                const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                uint32_t h[4], l[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = v[2 * j] * scale, y = v[2 * j + 1] * scale;
                    const __half2 q = __floats2half2_rn(x, y);
                    h[j] = *reinterpret_cast<const uint32_t*>(&q);
                    l[j] = pack2<false>(x - __low2float(q), y - __high2float(q));
                }
                hi = make_uint4(h[0], h[1], h[2], h[3]);
                lo = make_uint4(l[0], l[1], l[2], l[3]);
            } else {
                hi = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + at);
            }
        }
        *reinterpret_cast<uint4*>(dst + r * ld + c) = hi;
        if (kF32) *reinterpret_cast<uint4*>(dst + (rows_pad + r) * ld + c) = lo;
    }
}

// Gathers rows into the contraction's operand: [rows_pad][ld] 16-bit, a copy
// of bf16 values, or two f16 planes of a Float32 value times 2^q (hi rounded
// to nearest, lo the rest).  Rows past the ones that count are zero.
template <bool kF32>
__global__ void pack_kernel(const void* src, int64_t rows, int64_t cols, int64_t sr, int64_t sc, const int* row_map,
                            const HeadState* state, int use_count, int scale_of, uint16_t* dst, int64_t ld,
                            int64_t rows_pad) {
    __shared__ float tile[32][33];
    pdl_enter();
    const int64_t valid = use_count ? min(rows, int64_t(state->count)) : rows;
    const bool twice = !kF32 && use_count && state->few(0);  // the rows again for their gradients' remainders
    const float scale = kF32 ? pow2i(scale_exponent(state->amax[scale_of])) : 1.0f;
    const int64_t r0 = int64_t(blockIdx.x) * 32, c0 = int64_t(blockIdx.y) * 32;
    const bool by_rows = sr == 1 && sc != 1;
    const int x = threadIdx.x & 31, y0 = threadIdx.x >> 5;
    for (int y = y0; y < 32; y += 8) {
        int64_t r = r0 + (by_rows ? x : y);
        const int64_t c = c0 + (by_rows ? y : x);
        if (twice && r >= kFewRows) r -= kFewRows;
        float v = 0.0f;
        if (r < valid && c < cols) {
            const int64_t at = (row_map ? int64_t(row_map[r]) : r) * sr + c * sc;
            v = kF32 ? static_cast<const float*>(src)[at] : __bfloat162float(static_cast<const __nv_bfloat16*>(src)[at]);
        }
        tile[by_rows ? x : y][by_rows ? y : x] = v;
    }
    __syncthreads();
    for (int y = y0; y < 32; y += 8) {
        const int64_t r = r0 + y, c = c0 + x;
        if (r >= rows_pad || c >= ld) continue;
        const float v = tile[y][x];
        if (kF32) {
            const float s = v * scale;
            const __half hi = __float2half_rn(s);
            dst[r * ld + c] = __half_as_ushort(hi);
            dst[(rows_pad + r) * ld + c] = __half_as_ushort(__float2half_rn(s - __half2float(hi)));
        } else {
            const __nv_bfloat16 b = __float2bfloat16_rn(v);
            dst[r * ld + c] = __bfloat16_as_ushort(b);
        }
    }
}

// ---- after the forward ---------------------------------------------------------

struct MergeArgs {
    const float4* partial;
    int tiles, rows_pad;
    int64_t row0, T, V;      // compact rows [row0, T)
    const HeadState* state;
    const int* row_map;
    const int* targets;
    int ignore_index;
    const float* entropy;    // distillation, or null
    float factor;            // f
    float* row_loss;         // compact
    float* lse2;             // compact
    float* loss;             // per row, or null
    float* lse;              // per row, or null
};

// 32 rows x 8 slices of the tiles per CTA.
__global__ void __launch_bounds__(256) merge_kernel(const MergeArgs a) {
    __shared__ float4 part[8][32];
    pdl_enter();
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t i = a.row0 + int64_t(blockIdx.x) * 32 + lane;
    const int count = a.state->count;
    float ref = -INFINITY, sum = 0.0f, dot = 0.0f;
    if (i < count) {
        for (int t = slice; t < a.tiles; t += 8) {
            const float4 p = a.partial[int64_t(t) * a.rows_pad + i];
            const float next = fmaxf(ref, p.x), base = next == -INFINITY ? 0.0f : next;
            sum = sum * ex2(ref - base) + p.y * ex2(p.x - base);
            ref = next;
            dot += p.z;
        }
    }
    part[slice][lane] = make_float4(ref, sum, dot, 0.0f);
    __syncthreads();
    if (slice || i >= a.T) return;
    const int64_t row = a.row_map[i];
    if (i >= count) {
        float v = 0.0f;
        if (a.targets && a.targets[row] != a.ignore_index) v = NAN;  // a target outside the vocabulary
        if (a.loss) a.loss[row] = v;
        if (a.lse) a.lse[row] = 0.0f;
        return;
    }
    for (int s = 1; s < 8; ++s) {
        const float4 p = part[s][lane];
        const float next = fmaxf(ref, p.x), base = next == -INFINITY ? 0.0f : next;
        sum = sum * ex2(ref - base) + p.y * ex2(p.x - base);
        ref = next;
        dot += p.z;
    }
    const float l2 = ref + log2f(sum);
    const float v = a.factor * ((a.entropy ? a.entropy[i] : 0.0f) + (l2 - dot) * kLn2);
    a.lse2[i] = l2;
    a.row_loss[i] = v;
    if (a.loss) a.loss[row] = v;
    if (a.lse) a.lse[row] = l2 * kLn2;
}

// loss = mean of the compact rows' losses, summed in a fixed order.
__global__ void __launch_bounds__(1024) mean_kernel(const float* row_loss, const HeadState* state, float* loss) {
    __shared__ float part[32];
    pdl_enter();
    const int n = state->count;
    float s = 0.0f;
    for (int i = threadIdx.x; i < n; i += 1024) s += row_loss[i];
    s = warp_sum(s);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = warp_sum(part[threadIdx.x]);
        if (threadIdx.x == 0) *loss = state->bad ? NAN : s / float(n);
    }
}

// The kept exponentials of the logits become their gradient, in place:
// exp2(k2 z - ref) 2^(ref - lse2) is the softmax, and the target entries are
// written from their own Float32 logits (where the softmax is near p, the
// stored 11 bits of it would not be enough).  A CTA takes kScaleCols columns of
// a row; a thread 8 columns (bf16), a half warp 32 columns (Float32: hi and lo
// values replace the 64-column block they were computed from).
constexpr int kScaleCols = 8192;
struct ScaleArgs {
    uint16_t* grad;
    int64_t ld_grad, V;
    const float4* partial;
    int tile_n;              // columns of a tile; its halves start at 0 and 128
    int rows_pad, row0;
    const HeadState* state;
    const float* lse2;
    const float* coef;
    const int* ent_idx;
    const float* ent_p;
    const float* ent_s;
    int ent_k;
};
template <bool kF32>
__global__ void __launch_bounds__(256) scale_kernel(const ScaleArgs a) {
    __shared__ float factor[kScaleCols / 64];
    pdl_enter();
    // the last rows first: they are the ones the contraction left in L2, and the
    // next one starts with the first
    const int64_t i = int64_t(gridDim.x) - 1 - blockIdx.x;
    if (i >= a.state->count - a.row0) return;
    const int64_t c0 = int64_t(blockIdx.y) * kScaleCols;
    const int64_t c1 = min(c0 + kScaleCols, a.V);
    const float lse2 = a.lse2[i];
    const float coef = a.coef[i] * (kF32 ? pow2i(scale_exponent(a.state->amax[2])) : 1.0f);
    for (int64_t b = c0 + threadIdx.x * 64; b < c1; b += 256 * 64) {  // tiles are whole 64-column blocks
        const int64_t tile = b / a.tile_n, half = tile * 2 + (b - tile * a.tile_n >= 128);
        const float ref = a.partial[half * a.rows_pad + i].x;
        // (a half tile of nothing but -inf stored zeros)
        factor[(b - c0) / 64] = ref == -INFINITY ? 0.0f : ex2(ref - lse2) * coef * (kF32 ? 1.0f : 1.0f / 32768.0f);
    }
    __syncthreads();
    uint16_t* row = a.grad + i * a.ld_grad;
    const bool few = !kF32 && a.state->few(a.row0);
    uint16_t* rest = row + kFewRows * a.ld_grad;
    if (kF32) {
        const int lane = threadIdx.x & 31;
        for (int64_t b = c0 + (threadIdx.x >> 5) * 64; b < c1; b += 8 * 64) {
            float2 v = reinterpret_cast<const float2*>(row + 2 * b)[lane];
            const float f = factor[(b - c0) / 64];
            v.x = b + 2 * lane < a.V ? v.x * f : 0.0f;
            v.y = b + 2 * lane + 1 < a.V ? v.y * f : 0.0f;
            const __half2 hi = __floats2half2_rn(v.x, v.y);
            const __half2 lo = __floats2half2_rn(v.x - __low2float(hi), v.y - __high2float(hi));
            __syncwarp();
            reinterpret_cast<__half2*>(row + 2 * b)[lane] = hi;
            reinterpret_cast<__half2*>(row + 2 * b + 64)[lane] = lo;
            __syncwarp();
        }
    } else {
        for (int64_t c = c0 + threadIdx.x * 8; c < c1; c += 256 * 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(row + c);
            const float f = factor[(c - c0) / 64];
            const uint32_t e[4] = {v.x, v.y, v.z, v.w};
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 g = __half22float2(*reinterpret_cast<const __half2*>(&e[j]));
                g.x *= f;
                g.y *= f;
                const __nv_bfloat162 h = __floats2bfloat162_rn(g.x, g.y);
                hi[j] = *reinterpret_cast<const uint32_t*>(&h);
                lo[j] = pack2<true>(g.x - __low2float(h), g.y - __high2float(h));
            }
            *reinterpret_cast<uint4*>(row + c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if (few) *reinterpret_cast<uint4*>(rest + c) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
    __syncthreads();  // the entries overwrite what the loop above wrote
    for (int k = threadIdx.x; k < a.ent_k; k += 256) {
        const int64_t at = i * a.ent_k + k;
        const int col = a.ent_idx[at];
        if (col < c0 || col >= c1 || (k > 0 && a.ent_idx[at - 1] == col)) continue;
        float p = a.ent_p ? a.ent_p[at] : 1.0f;
        for (int j = 1; k + j < a.ent_k && a.ent_idx[at + j] == col; ++j) p += a.ent_p[at + j];
        const float g = (ex2(a.ent_s[at] - lse2) - p) * coef;
        if (kF32) {
            uint16_t* d = row + (col & ~63) * int64_t(2) + (col & 63);
            const __half hi = __float2half_rn(g);
            d[0] = __half_as_ushort(hi);
            d[64] = __half_as_ushort(__float2half_rn(g - __half2float(hi)));
        } else {
            const __nv_bfloat16 hi = __float2bfloat16_rn(g);
            row[col] = __bfloat16_as_ushort(hi);
            if (few) rest[col] = __bfloat16_as_ushort(__float2bfloat16_rn(g - __bfloat162float(hi)));
        }
    }
}

// Result rows from the fp32 sums of the K walk's parts, added in order, to
// their places; with by_count, zeros in the rows that do not count.
struct SlotsArgs {
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
template <bool kF32>
__global__ void __launch_bounds__(256) sum_slots_kernel(const SlotsArgs a) {
    pdl_enter();
    const int splits = a.splits > 0 ? a.splits : a.state->dh_splits;
    const int64_t summed = a.by_count ? min(a.rows, int64_t(a.state->rows(a.row0))) : a.rows;
    const bool few = !kF32 && a.by_count && a.state->few(a.row0);  // their remainders are further rows
    const Walk walk(few ? a.state->rows_and_rest(a.row0, true) : int(summed), int((a.cols + kBN - 1) / kBN), a.tile_m, a.workers, splits);
    const int64_t per_row = (a.cols + 3) / 4;
    for (int64_t u = int64_t(blockIdx.x) * 256 + threadIdx.x; u < a.rows * per_row; u += int64_t(gridDim.x) * 256) {
        const int64_t m = u / per_row, c = (u - m * per_row) * 4;
        const float* p = a.sums + c;  // ld is whole groups of four
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (m < summed) {
            const int tile = walk.tile_of(int(m) / a.tile_m, int(c) / kBN);
            const int parts = tile < walk.whole ? 1 : splits;
            for (int rest = 0; rest <= (few ? kFewRows : 0); rest += kFewRows) {
#pragma unroll 4
                for (int k = 0; k < parts; ++k) {
                    const float4 v =
                        *reinterpret_cast<const float4*>(p + int64_t(walk.sum_row(k, int(m) + rest)) * a.ld);
                    s.x += v.x;
                    s.y += v.y;
                    s.z += v.z;
                    s.w += v.w;
                }
            }
        }
        const int64_t at = (a.row_map ? int64_t(a.row_map[m]) : m) * a.dst_row + c * a.dst_col;
        const float r[4] = {s.x, s.y, s.z, s.w};
        if (a.vec && c + 4 <= a.cols) {
            if (kF32) *reinterpret_cast<float4*>(static_cast<float*>(a.dst) + at) = s;
            else
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.dst) + at) =
                    make_uint2(pack2<true>(s.x, s.y), pack2<true>(s.z, s.w));
            continue;
        }
        for (int j = 0; j < 4 && c + j < a.cols; ++j) {
            if (kF32) static_cast<float*>(a.dst)[at + j * a.dst_col] = r[j];
            else static_cast<__nv_bfloat16*>(a.dst)[at + j * a.dst_col] = __float2bfloat16_rn(r[j]);
        }
    }
}

// ---- host ----------------------------------------------------------------------

// 2-D map over rows x cols 16-bit elements (pitch ld elements), 64 x box_rows
// boxes, 128-byte swizzle; what lies outside reads as zero.
int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, uint32_t box_rows) {
    auto fn = tensor_map_encoder();
    if (!fn) return fail(SW_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(ld * 2)};
    cuuint32_t box[2] = {(cuuint32_t)kBK, box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(SW_ERR_CUDA, "cuTensorMapEncodeTiled (linear head) failed (%d)", (int)r);
    return SW_OK;
}

// A contraction operand: `rows` x `cols` 16-bit elements in memory, pitch ld
// (every plane of them), and where its lo plane lies.
struct Operand {
    const uint16_t* ptr;
    int64_t rows, cols, ld;
    Plane plane;
};

int64_t round_up(int64_t x, int64_t q) { return (x + q - 1) / q * q; }

int device_sms() {
    static int sms[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        sms[dev] = 148;
    return sms[dev];
}

// How a contraction is spread over the SMs: the tile shape and the parts of the
// K walk.
struct Spread {
    int shape;
    int splits;
};
// `sum_us`: what it costs more to go through fp32 sums when nothing else asks
// for them.
Spread choose_spread(int64_t M, int64_t N, int64_t K, int terms, int tallest, bool may_split, float sum_us = 0.0f) {
    Spread best{kSingle, 1};
    float best_us = 1e30f;
    for (int shape = tallest; shape >= kSingle; --shape)
        for (int s = 1; s <= (may_split ? kMaxParts : 1); ++s) {
            const float us = spread_cost(M, N, K, terms, shape, device_sms(), s) + (s > 1 ? sum_us : 0.0f);
            if (us < best_us * 0.97f) {
                best_us = us;
                best = Spread{shape, s};
            }
        }
    return best;
}

// Rows of fp32 sums that the parts of any row count up to M may take: all rows,
// and those of the parts past the first, of at most two tiles per worker where
// the tiles do not fill a wave, else of the row groups that the last wave
// reaches.
int64_t sum_rows(int64_t M, int64_t N, int shape) {
    const int64_t cols = (N + kBN - 1) / kBN, tile_m = shape_rows(shape), all = round_up(M, tile_m);
    const int64_t workers = shape_workers(shape, device_sms()), group = 2048 / tile_m;
    const int64_t few = (2 * workers / cols + 1) * tile_m;
    const int64_t tail = std::min(all, (workers / (group * cols) + 2) * group * tile_m) * (kMaxTailParts - 1);
    return all + std::max(few, tail);
}

// Where a contraction writes through its output map: 16-bit or Float32 values,
// in boxes of 128 bytes x 32 rows.
struct Target {
    const void* ptr;         // null: no map
    int64_t rows, cols, ld;  // elements
    bool f32;
};

int make_target_map(CUtensorMap* map, const Target& t) {
    auto fn = tensor_map_encoder();
    if (!fn) return fail(SW_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[2] = {(cuuint64_t)t.cols, (cuuint64_t)t.rows};
    cuuint64_t strides[1] = {(cuuint64_t)(t.ld * (t.f32 ? 4 : 2))};
    cuuint32_t box[2] = {t.f32 ? 32u : 64u, 32};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, t.f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2,
                    const_cast<void*>(t.ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(SW_ERR_CUDA, "cuTensorMapEncodeTiled (linear head result) failed (%d)", (int)r);
    return SW_OK;
}

template <int kShape, bool kBf16, bool kAMn, bool kBMn, int kEpi>
int launch_gemm(const Operand& a, const Operand& b, const Target& c, const GemmArgs& args, cudaStream_t stream) {
    using Cf = Cfg<kShape>;
    constexpr bool kPair = Cf::kPair;
    const int64_t tiles = int64_t((args.M + Cf::kTileM - 1) / Cf::kTileM) * ((args.N + args.tile_n - 1) / args.tile_n);
    if (tiles == 0) return SW_OK;
    CUtensorMap ma, mb, mc;
    int rc = make_map(&ma, a.ptr, a.rows, a.cols, a.ld, kAMn ? kBK : kBM);
    if (rc != SW_OK) return rc;
    rc = make_map(&mb, b.ptr, b.rows, b.cols, b.ld, kBMn ? kBK : kPair ? Cf::kBRows : args.tile_n);
    if (rc != SW_OK) return rc;
    memset(&mc, 0, sizeof(mc));
    if (c.ptr && (rc = make_target_map(&mc, c)) != SW_OK) return rc;
    auto kernel = head_gemm_kernel<kShape, kBf16, kAMn, kBMn, kEpi>;
    SW_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cf::kSmemBytes),
                "linear head smem");
    constexpr int kCtas = kPair ? 2 : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kCtas * (unsigned)(args.splits == 1 ? std::min<int64_t>(tiles, device_sms() / kCtas) : device_sms() / kCtas));
    cfg.blockDim = dim3(Cf::kThreads);
    cfg.dynamicSmemBytes = Cf::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kCtas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kPair ? 2 : 1;
    SW_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ma, mb, mc, args), "linear head contraction");
    return SW_OK;
}

template <bool kBf16, bool kAMn, bool kBMn, int kEpi>
int gemm(const Operand& a, const Operand& b, const Target& c, GemmArgs args, int shape, cudaStream_t stream) {
    args.terms = kBf16 ? 1 : 3;
    args.pa = a.plane;
    args.pb = b.plane;
    if (kEpi != kEpiOut) args.splits = 1;
    if (kEpi != kEpiLse || shape != kSingle) args.tile_n = kBN;
    if (shape == kSingle) return launch_gemm<kSingle, kBf16, kAMn, kBMn, kEpi>(a, b, c, args, stream);
    // results summed in registers (Float32, and the statistics) have no tall tile,
    // and the logits' gradient has too much to do after a tile (4096 x 32000, dim
    // 1024 / 2048 / 4096: 242 / 395 / 719 us against 201 / 362 / 695)
    constexpr int kTallest = kBf16 && kEpi == kEpiOut ? kTall : kPair2;
    return shape == kTall ? launch_gemm<kTallest, kBf16, kAMn, kBMn, kEpi>(a, b, c, args, stream)
                          : launch_gemm<kPair2, kBf16, kAMn, kBMn, kEpi>(a, b, c, args, stream);
}

struct Bump {
    uint8_t* base;
    int64_t used;
    template <class T>
    T* take(int64_t n) {
        used = (used + 255) / 256 * 256;
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used += n * (int64_t)sizeof(T);
        return p;
    }
};

struct Call {
    const sw_linear_head* plan;
    const void* h;
    const void* w;
    const int32_t* targets;
    int32_t ignore_index;
    const int32_t* teacher_index;
    const float* teacher_logits;
    int top_k;
    float scale, factor;     // c, f
    float* loss;
    float* lse;
    const float* upstream;
    void* dh;
    void* dw;
};

// Everything the call needs in device memory, as offsets into one block.
struct Layout {
    HeadState* state;
    uint8_t* flags;
    int* row_map;
    int* ent_idx;
    float* ent_p;
    float* entropy;
    uint16_t* offs;
    float* coef;
    float* lse2;
    float* row_loss;
    float* ent_s;
    uint16_t* hc;
    float4* partial;
    float* dh_sums;
    float* dw_sums;
    uint16_t* wp;
    uint16_t* grad;
};

struct Shape {
    int64_t T, D, V, rows_pad, ld_h, ld_w;
    int64_t half_tiles;      // 128-column pieces of the vocabulary, each with its statistics
    bool f32, pack_w, grads;
    int planes;
    // Gradients: `keep`: the forward's exponentials of `rows` compact rows at a
    // time stay in the workspace and become the logits' gradient.  Otherwise
    // the logits are computed again, `piece` columns of the vocabulary at a
    // time.  Packed weights are laid out `piece` columns at a time too.
    bool keep;
    int64_t rows, piece;
    int tile_n;              // columns of a logits tile
    int logits_shape, dh_shape;
    Spread dw;
    // rows of fp32 sums of each gradient (0: it is written at once); dh's rows
    // are always put in place from sums, whose parts are chosen on the device
    int64_t dh_sum_rows, dw_sum_rows, ld_acc;
};

Layout lay_out(Bump& b, const Call& c, const Shape& s) {
    Layout l;
    memset(&l, 0, sizeof(l));
    const int64_t K = c.targets ? 1 : c.top_k;
    l.state = b.take<HeadState>(1);
    l.row_map = b.take<int>(s.T);
    l.ent_idx = b.take<int>(s.rows_pad * K);
    if (!c.targets) {
        l.flags = b.take<uint8_t>(s.T);
        l.ent_p = b.take<float>(s.rows_pad * K);
        l.entropy = b.take<float>(s.rows_pad);
        l.offs = b.take<uint16_t>(s.rows_pad * ((s.V + kEntryTile - 1) / kEntryTile + 1));
    }
    l.coef = b.take<float>(s.rows_pad);
    l.lse2 = b.take<float>(s.rows_pad);
    l.row_loss = b.take<float>(s.rows_pad);
    l.hc = b.take<uint16_t>(s.planes * s.rows_pad * s.ld_h);
    if (c.loss) l.partial = b.take<float4>(s.half_tiles * s.rows_pad);
    if (s.keep) l.ent_s = b.take<float>(s.rows_pad * K);
    if (s.dh_sum_rows) l.dh_sums = b.take<float>(s.dh_sum_rows * s.ld_acc);
    if (s.dw_sum_rows) l.dw_sums = b.take<float>(s.dw_sum_rows * s.ld_acc);
    if (s.pack_w) l.wp = b.take<uint16_t>(s.planes * round_up(s.piece, kBK) * s.ld_w);
    if (s.grads) l.grad = b.take<uint16_t>(s.planes * s.rows * round_up(s.piece, 64));
    return l;
}

template <bool kF32>
int run(const Call& c, const Shape& s, const Layout& l, cudaStream_t stream) {
    const sw_linear_head& p = *c.plan;
    constexpr bool kBf16 = !kF32;
    const int esize = kF32 ? 4 : 2, terms = kF32 ? 3 : 1;
    SW_CUDA_TRY(cudaMemsetAsync(l.state, 0, sizeof(HeadState), stream), "linear head state");
    if (!c.targets)
        SW_CUDA_TRY(launch_pdl(teacher_flags_kernel, dim3((unsigned)std::max<int64_t>((s.T + 7) / 8, 1)), dim3(256), 0, stream,
                               c.teacher_index, c.teacher_logits, s.T, c.top_k, s.V, l.flags),
                    "teacher rows");
    RowsArgs ra;
    memset(&ra, 0, sizeof(ra));
    ra.targets = c.targets;
    ra.ignore_index = c.ignore_index;
    ra.flags = l.flags;
    ra.T = s.T;
    ra.V = s.V;
    ra.upstream = c.upstream;
    ra.mean = p.reduction == SW_HEAD_MEAN;
    ra.factor = c.scale * c.factor;
    ra.lse = c.loss ? nullptr : c.lse;
    ra.row_map = l.row_map;
    ra.ent_idx = l.ent_idx;
    ra.coef = s.grads ? l.coef : nullptr;
    ra.lse2 = l.lse2;
    ra.state = l.state;
    ra.dh_rows = s.rows;
    ra.dh_cols = s.D;
    ra.dh_k = std::min(s.piece, s.V);
    ra.dh_shape = s.dh_shape;
    ra.sms = device_sms();
    ra.terms = terms;
    SW_CUDA_TRY(launch_pdl(rows_kernel, dim3(1), dim3(1024), 0, stream, ra), "linear head rows");
    if (!c.targets)
        SW_CUDA_TRY(launch_pdl(teacher_sort_kernel, dim3((unsigned)std::max<int64_t>((s.T + 3) / 4, 1)), dim3(128), 0, stream,
                               c.teacher_index, c.teacher_logits, c.top_k, s.V, c.scale, l.row_map, l.state,
                               (int)s.rows_pad, (int)((s.V + kEntryTile - 1) / kEntryTile), l.ent_idx, l.ent_p,
                               l.entropy, l.offs),
                    "teacher entries");
    // rows of `cols` elements that the vector kernels can read
    auto whole_rows = [&](const void* x, int64_t cols, int64_t sr, int64_t sc) {
        return sc == 1 && cols % 8 == 0 && sr * esize % 16 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    };
    const unsigned fill = (unsigned)(8 * device_sms());
    auto amax = [&](const void* x, int64_t rows, int64_t sr, int64_t sc, const int* map, const HeadState* count,
                    uint32_t* out) -> int {
        SW_CUDA_TRY(launch_pdl(amax_kernel, dim3(std::min<unsigned>(fill, (unsigned)((std::max(rows, s.D) + 7) / 8))),
                               dim3(256), 0, stream, (const float*)x, rows, s.D, sr, sc,
                               (int)whole_rows(x, s.D, sr, sc), map, count, out),
                    "linear head scale");
        return SW_OK;
    };
    auto pack = [&](const void* x, int64_t rows, int64_t sr, int64_t sc, const int* map, int use_count, int scale_of,
                    uint16_t* dst, int64_t rows_pad) -> int {
        if (whole_rows(x, s.D, sr, sc)) {
            const int64_t units = rows_pad * (s.D / 8);
            SW_CUDA_TRY(launch_pdl(pack_rows_kernel<kF32>, dim3((unsigned)std::min<int64_t>((units + 255) / 256, fill)),
                                   dim3(256), 0, stream, x, rows, s.D, sr, map, l.state, use_count, scale_of, dst,
                                   s.ld_h, rows_pad),
                        "linear head operand");
        } else {
            SW_CUDA_TRY(launch_pdl(pack_kernel<kF32>,
                                   dim3((unsigned)((rows_pad + 31) / 32), (unsigned)((s.ld_h + 31) / 32)), dim3(256), 0,
                                   stream, x, rows, s.D, sr, sc, map, l.state, use_count, scale_of, dst, s.ld_h,
                                   rows_pad),
                        "linear head operand");
        }
        return SW_OK;
    };
    int rc;
    if (kF32) {
        if ((rc = amax(c.h, s.T, p.h_row, p.h_col, l.row_map, l.state, &l.state->amax[0])) != SW_OK) return rc;
        if ((rc = amax(c.w, s.V, p.w_row, p.w_col, nullptr, nullptr, &l.state->amax[1])) != SW_OK) return rc;
    }
    if ((rc = pack(c.h, s.T, p.h_row, p.h_col, l.row_map, 1, 0, l.hc, s.rows_pad)) != SW_OK) return rc;
    const Plane dense{kBK, 0, 0};
    // rows [r0, r0 + n) of the gathered states
    auto states = [&](int64_t r0, int64_t n) {
        return Operand{l.hc + r0 * s.ld_h, kF32 ? s.rows_pad + n : n, s.D, s.ld_h, Plane{kBK, 0, (int)s.rows_pad}};
    };
    const int64_t ld_grad = s.planes * round_up(s.piece, 64);

    GemmArgs g;
    memset(&g, 0, sizeof(g));
    g.state = l.state;
    g.logit_scale = c.scale;
    g.ent_p = l.ent_p;
    g.ent_k = c.targets ? 1 : c.top_k;
    g.rows_pad = (int)s.rows_pad;
    g.tile_n = s.tile_n;
    const Target grad_out{l.grad, s.rows, ld_grad, ld_grad, false}, none{nullptr, 0, 0, 0, false};

    // the weights of columns [v0, v0 + n): in place, or packed into the workspace
    int64_t packed = -1;
    auto weights = [&](int64_t v0, int64_t n, Operand* out) -> int {
        const uint8_t* at = static_cast<const uint8_t*>(c.w) + v0 * p.w_row * esize;
        if (!s.pack_w) {
            *out = Operand{reinterpret_cast<const uint16_t*>(at), n, s.D, p.w_row, dense};
            return SW_OK;
        }
        // zero rows up to whole K stages: a tail of G's zeros must not meet the next plane
        const int64_t rows = round_up(n, kBK);
        if (packed != v0) {
            const int rc = pack(at, n, p.w_row, p.w_col, nullptr, 0, 1, l.wp, rows);
            if (rc != SW_OK) return rc;
        }
        packed = v0;
        *out = Operand{l.wp, s.planes * rows, s.D, s.ld_w, Plane{kBK, 0, (int)rows}};
        return SW_OK;
    };
    // logits of compact rows [r0, r0 + n) and columns [v0, v0 + nv)
    auto logits = [&](int64_t r0, int64_t n, int64_t v0, int64_t nv) {
        GemmArgs a = g;
        a.M = (int)n;
        a.N = (int)nv;
        a.K = (int)s.D;
        a.count_is = kCountM;
        a.row0 = (int)r0;
        a.scale_a = kF32 ? 0 : -1;
        a.scale_b = kF32 ? 1 : -1;
        a.v0 = v0;
        a.half0 = (int)(v0 / kBN * 2);
        a.ent_idx = l.ent_idx + r0 * g.ent_k;
        a.ent_p = l.ent_p ? l.ent_p + r0 * g.ent_k : nullptr;
        a.offs = l.offs ? l.offs + r0 : nullptr;
        a.partial = l.partial + r0;
        a.lse2 = l.lse2 + r0;
        a.coef = l.coef + r0;
        return a;
    };
    auto merge = [&](int64_t r0, int64_t n) -> int {
        MergeArgs m;
        memset(&m, 0, sizeof(m));
        m.partial = l.partial;
        m.tiles = (int)s.half_tiles;
        m.rows_pad = (int)s.rows_pad;
        m.row0 = r0;
        m.T = std::min(s.T, r0 + n);
        m.V = s.V;
        m.state = l.state;
        m.row_map = l.row_map;
        m.targets = c.targets;
        m.ignore_index = c.ignore_index;
        m.entropy = l.entropy;
        m.factor = c.factor;
        m.row_loss = l.row_loss;
        m.lse2 = l.lse2;
        m.loss = p.reduction == SW_HEAD_MEAN ? nullptr : c.loss;
        m.lse = c.lse;
        SW_CUDA_TRY(launch_pdl(merge_kernel, dim3((unsigned)std::max<int64_t>((n + 31) / 32, 1)), dim3(256), 0, stream,
                               m),
                    "linear head loss");
        return SW_OK;
    };
    // dh of compact rows [r0, r0 + n) += G[:, 0..nv) w;  dw of columns [v0, v0 + nv) += G^T h
    auto gradients = [&](int64_t r0, int64_t n, int64_t v0, int64_t nv, const Operand& w, bool first_v, bool last_v,
                         bool first_r, bool last_r) -> int {
        const Plane gp = kF32 ? Plane{2 * kBK, kBK, 0} : dense;
        const Operand gr{l.grad, s.rows, kF32 ? 2 * round_up(nv, 64) : nv, ld_grad, gp};
        GemmArgs a = g;
        a.row0 = (int)r0;
        auto finish = [&](float* sums, int splits, int shape, int64_t rows, bool by_count, const int* row_map,
                          void* dst, int64_t dst_row, int64_t dst_col) -> int {
            SlotsArgs sa;
            memset(&sa, 0, sizeof(sa));
            sa.sums = sums;
            sa.ld = s.ld_acc;
            sa.splits = splits;
            sa.tile_m = shape_rows(shape);
            sa.workers = shape_workers(shape, device_sms());
            sa.rows = rows;
            sa.cols = s.D;
            sa.state = l.state;
            sa.by_count = by_count;
            sa.row0 = (int)r0;
            sa.row_map = row_map;
            sa.dst = dst;
            sa.dst_row = dst_row;
            sa.dst_col = dst_col;
            sa.vec = dst_col == 1 && dst_row % 4 == 0 && (reinterpret_cast<uintptr_t>(dst) & (4 * esize - 1)) == 0;
            const int64_t units = rows * (s.ld_acc / 4);
            SW_CUDA_TRY(launch_pdl(sum_slots_kernel<kF32>, dim3((unsigned)std::min<int64_t>((units + 255) / 256, fill)),
                                   dim3(256), 0, stream, sa),
                        "linear head sums");
            return SW_OK;
        };
        if (c.dh && n > 0) {
            a.M = (int)n;
            a.N = (int)s.D;
            a.K = (int)nv;
            a.count_is = kCountM;
            a.scale_a = kF32 ? 2 : -1;
            a.scale_b = kF32 ? 1 : -1;
            a.splits = 0;
            a.sums = 1;
            a.first = first_v;
            const Target out{l.dh_sums, s.dh_sum_rows, s.ld_acc, s.ld_acc, true};
            int rc = gemm<kBf16, false, true, kEpiOut>(gr, w, out, a, s.dh_shape, stream);
            if (rc == SW_OK && last_v)
                rc = finish(l.dh_sums, 0, s.dh_shape, n, true, l.row_map + r0, c.dh, p.dh_row, p.dh_col);
            if (rc != SW_OK) return rc;
        }
        if (c.dw) {
            uint8_t* dst = static_cast<uint8_t*>(c.dw) + v0 * p.dw_row * esize;
            a.M = (int)nv;
            a.N = (int)s.D;
            a.K = (int)n;
            a.count_is = kCountK;
            a.scale_a = kF32 ? 2 : -1;
            a.scale_b = kF32 ? 0 : -1;
            a.splits = s.dw.splits;
            a.sums = s.dw_sum_rows > 0;
            a.first = first_r;
            const Target out = a.sums ? Target{l.dw_sums, s.dw_sum_rows, s.ld_acc, s.ld_acc, true}
                                      : Target{dst, nv, s.D, p.dw_row, kF32};
            int rc = gemm<kBf16, true, true, kEpiOut>(gr, states(r0, round_up(std::max<int64_t>(n, 1), kBM)), out, a,
                                                      s.dw.shape, stream);
            if (rc == SW_OK && a.sums && last_r)
                rc = finish(l.dw_sums, s.dw.splits, s.dw.shape, nv, false, nullptr, dst, p.dw_row, p.dw_col);
            if (rc != SW_OK) return rc;
        }
        return SW_OK;
    };
    auto mean = [&]() -> int {
        if (c.loss && p.reduction == SW_HEAD_MEAN)
            SW_CUDA_TRY(launch_pdl(mean_kernel, dim3(1), dim3(1024), 0, stream, l.row_loss, l.state, c.loss),
                        "linear head mean loss");
        return SW_OK;
    };
    if (s.keep) {
        Operand w;
        if ((rc = weights(0, s.V, &w)) != SW_OK) return rc;
        for (int64_t r0 = 0; r0 == 0 || r0 < s.T; r0 += s.rows) {
            const int64_t n = std::min(s.rows, s.T - r0);
            GemmArgs a = logits(r0, n, 0, s.V);
            a.keep = 1;
            a.ent_s = l.ent_s + r0 * g.ent_k;
            rc = gemm<kBf16, false, false, kEpiLse>(states(r0, round_up(std::max<int64_t>(n, 1), kBM)), w, grad_out, a,
                                                    s.logits_shape, stream);
            if (rc != SW_OK) return rc;
            if ((rc = merge(r0, n)) != SW_OK) return rc;
            ScaleArgs sc;
            memset(&sc, 0, sizeof(sc));
            sc.grad = l.grad;
            sc.ld_grad = ld_grad;
            sc.V = s.V;
            sc.partial = a.partial;
            sc.tile_n = s.tile_n;
            sc.rows_pad = (int)s.rows_pad;
            sc.row0 = (int)r0;
            sc.state = l.state;
            sc.lse2 = a.lse2;
            sc.coef = a.coef;
            sc.ent_idx = a.ent_idx;
            sc.ent_p = a.ent_p;
            sc.ent_s = a.ent_s;
            sc.ent_k = g.ent_k;
            if (n > 0)
                SW_CUDA_TRY(launch_pdl(scale_kernel<kF32>,
                                       dim3((unsigned)n, (unsigned)((s.V + kScaleCols - 1) / kScaleCols)), dim3(256), 0,
                                       stream, sc),
                            "linear head logits' gradient");
            if ((rc = gradients(r0, n, 0, s.V, w, true, true, r0 == 0, r0 + s.rows >= s.T)) != SW_OK) return rc;
        }
        return mean();
    }
    if (c.loss) {
        const int64_t step = s.pack_w ? s.piece : s.V;
        for (int64_t v0 = 0; v0 < s.V; v0 += step) {
            const int64_t n = std::min(step, s.V - v0);
            Operand w;
            if ((rc = weights(v0, n, &w)) != SW_OK) return rc;
            rc = gemm<kBf16, false, false, kEpiLse>(states(0, s.rows_pad), w, none, logits(0, s.T, v0, n), s.logits_shape,
                                                    stream);
            if (rc != SW_OK) return rc;
        }
        if ((rc = merge(0, s.T)) != SW_OK) return rc;
        if ((rc = mean()) != SW_OK) return rc;
    }
    if (!s.grads) return SW_OK;
    for (int64_t v0 = 0; v0 < s.V; v0 += s.piece) {
        const int64_t n = std::min(s.piece, s.V - v0);
        Operand w;
        if ((rc = weights(v0, n, &w)) != SW_OK) return rc;
        rc = gemm<kBf16, false, false, kEpiGrad>(states(0, s.rows_pad), w, grad_out, logits(0, s.T, v0, n),
                                                 s.logits_shape, stream);
        if (rc != SW_OK) return rc;
        if ((rc = gradients(0, s.T, v0, n, w, v0 == 0, v0 + n == s.V, true, true)) != SW_OK) return rc;
    }
    return SW_OK;
}

// A matrix's strides must reach each element once (gradients) and fit 63 bits.
bool strides_ok(int64_t rows, int64_t cols, int64_t sr, int64_t sc, bool distinct) {
    if (sr < 0 || sc < 0) return false;
    const int64_t lim = int64_t(1) << 52;
    if ((rows > 1 && sr > lim / rows) || (cols > 1 && sc > lim / cols)) return false;
    if (!distinct) return true;
    if (rows > 1 && sr == 0) return false;
    if (cols > 1 && sc == 0) return false;
    if (rows == 1 || cols == 1) return true;
    return sr <= sc ? sc > (rows - 1) * sr : sr > (cols - 1) * sc;
}

int check_and_run(const char* name, Call& c, void* stream_ptr) {
    const sw_linear_head* p = c.plan;
    if (!p) return fail(SW_ERR_INVALID, "%s: null plan", name);
    if (p->dtype != SW_HEAD_F32 && p->dtype != SW_HEAD_BF16)
        return fail(SW_ERR_INVALID, "%s: unknown dtype %d", name, (int)p->dtype);
    if (p->reduction != SW_HEAD_NONE && p->reduction != SW_HEAD_MEAN)
        return fail(SW_ERR_INVALID, "%s: unknown reduction %d", name, (int)p->reduction);
    if (p->tokens < 0 || p->dim < 1 || p->vocab < 1)
        return fail(SW_ERR_INVALID, "%s: tokens must be >= 0, dim and vocab positive (got %lld, %lld, %lld)", name,
                    (long long)p->tokens, (long long)p->dim, (long long)p->vocab);
    const int64_t lim = int64_t(1) << 30;
    if (p->tokens > lim || p->dim > lim || p->vocab > lim)
        return fail(SW_ERR_UNSUPPORTED, "%s: extents above 2^30 are not supported", name);
    if (((p->tokens + kBM - 1) / kBM) * ((p->vocab + 63) / 64) > INT32_MAX ||
        ((p->vocab + kBM - 1) / kBM) * ((p->dim + 63) / 64) > INT32_MAX || (p->dim + 31) / 32 > 65535)
        return fail(SW_ERR_UNSUPPORTED, "%s: too many tiles", name);
    if (p->workspace_limit < 0) return fail(SW_ERR_INVALID, "%s: negative workspace limit", name);
    if (!(c.scale > 0.0f) || !std::isfinite(c.scale) || !std::isfinite(c.factor))
        return fail(SW_ERR_INVALID, "%s: the logit scale or temperature must be positive and finite", name);
    const bool grads = c.dh || c.dw;
    // (the vectors of no rows may be null)
    if (!c.loss && !grads && p->tokens == 0 && p->reduction == SW_HEAD_NONE) return ok();
    if (!c.loss && !grads) return fail(SW_ERR_INVALID, "%s: neither a loss nor a gradient is asked for", name);
    if (!c.loss && !c.lse && p->tokens > 0)
        return fail(SW_ERR_INVALID, "%s: a gradient without the loss needs the kept lse", name);
    const int64_t T = p->tokens, D = p->dim, V = p->vocab;
    if (T > 0 && !c.h) return fail(SW_ERR_INVALID, "%s: null states", name);
    if (!c.w) return fail(SW_ERR_INVALID, "%s: null weights", name);
    if (!strides_ok(T, D, p->h_row, p->h_col, false) || !strides_ok(V, D, p->w_row, p->w_col, false))
        return fail(SW_ERR_INVALID, "%s: bad strides of the states or weights", name);
    if (c.dh && !strides_ok(T, D, p->dh_row, p->dh_col, true))
        return fail(SW_ERR_INVALID, "%s: the strides of dh must reach every element once", name);
    if (c.dw && !strides_ok(V, D, p->dw_row, p->dw_col, true))
        return fail(SW_ERR_INVALID, "%s: the strides of dw must reach every element once", name);
    const uintptr_t align = p->dtype == SW_HEAD_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(c.h) | reinterpret_cast<uintptr_t>(c.w) | reinterpret_cast<uintptr_t>(c.dh) |
         reinterpret_cast<uintptr_t>(c.dw)) & align)
        return fail(SW_ERR_INVALID, "%s: a matrix is not aligned to its elements", name);
    if ((reinterpret_cast<uintptr_t>(c.loss) | reinterpret_cast<uintptr_t>(c.lse) |
         reinterpret_cast<uintptr_t>(c.upstream) | reinterpret_cast<uintptr_t>(c.targets) |
         reinterpret_cast<uintptr_t>(c.teacher_index) | reinterpret_cast<uintptr_t>(c.teacher_logits)) & 3)
        return fail(SW_ERR_INVALID, "%s: a vector is not aligned to its elements", name);
    cudaStream_t stream = (cudaStream_t)stream_ptr;

    Shape s;
    s.T = T;
    s.D = D;
    s.V = V;
    s.f32 = p->dtype == SW_HEAD_F32;
    s.planes = s.f32 ? 2 : 1;
    s.rows_pad = std::max<int64_t>(round_up(T, kBM), kBM);
    s.ld_h = s.ld_w = round_up(D, 8);
    s.grads = grads;
    s.ld_acc = round_up(D, 4);
    // weights are read in place when TMA can: bf16, unit stride, 16-byte rows
    s.pack_w = s.f32 || p->w_col != 1 || p->w_row % 8 != 0 || p->w_row < D ||
               (reinterpret_cast<uintptr_t>(c.w) & 15) != 0;
    const int64_t budget = p->workspace_limit > 0 ? p->workspace_limit : kDefaultWorkspace;
    const int64_t packed = s.pack_w ? s.planes * round_up(V, kBK) * s.ld_w * 2 : 0;
    const int64_t grad_row = s.planes * round_up(V, 256) * 2;
    const int terms = s.f32 ? 3 : 1;
    // One call for the loss and the gradients keeps the logits' exponentials
    // of as many rows as the workspace limit allows (6 T V D operations and one
    // more pass over them); from a kept lse, or where not even 1024 rows (or
    // all) fit, the logits are computed again (8 T V D).
    s.rows = s.rows_pad;
    s.keep = false;
    if (c.loss && grads && packed < budget) {
        const int64_t fit = (budget - packed) / grad_row / kBM * kBM;
        if (fit >= std::min<int64_t>(s.rows_pad, 1024)) {
            s.keep = true;
            const int64_t chunks = (s.rows_pad + fit - 1) / fit;
            s.rows = std::min(s.rows_pad, round_up((s.rows_pad + chunks - 1) / chunks, kBM));
        }
    }
    s.piece = round_up(V, 256);
    if (!s.keep) {
        // as wide as the limit allows, in whole 256-column tiles
        const int64_t per_column = (grads ? s.planes * s.rows_pad * 2 : 0) + (s.pack_w ? s.planes * s.ld_w * 2 : 0);
        if (per_column > 0) s.piece = std::min(s.piece, std::max<int64_t>(budget / per_column / 256 * 256, 256));
    }
    const int tallest = s.f32 ? kPair2 : kTall;
    s.logits_shape = choose_spread(std::min(s.rows, T), std::min(s.piece, V), D, terms, kPair2, false).shape;
    s.tile_n = kBN;
    if (s.logits_shape == kSingle && c.loss && (s.piece >= V || !s.pack_w)) {
        // few rows: a tile as narrow as fills the last wave (whole 64-column
        // blocks where the exponentials are kept, else whole MMA widths)
        const int q = s.keep ? 64 : 16, sms = device_sms();
        const int64_t row_tiles = (T + kBM - 1) / kBM;
        int64_t best = INT64_MAX;
        for (int t = kBN; t >= 128; t -= q) {
            const int64_t tiles = row_tiles * ((V + t - 1) / t), cost = (tiles + sms - 1) / sms * (t + 16);
            if (cost < best) {
                best = cost;
                s.tile_n = t;
            }
        }
    }
    s.half_tiles = (V + s.tile_n - 1) / s.tile_n * 2;
    s.dh_shape = kSingle;
    s.dw = Spread{kSingle, 1};
    s.dh_sum_rows = s.dw_sum_rows = 0;
    if (c.dh && T > 0) {
        const int64_t n = std::min(s.rows, T), nv = std::min(s.piece, V);
        s.dh_shape = choose_spread(n, D, nv, terms, tallest, true).shape;
        s.dh_sum_rows = sum_rows(n, D, s.dh_shape);
    }
    if (c.dw) {
        const int64_t n = std::min(s.rows, T), nv = std::min(s.piece, V);
        // written at once through TMA where that can describe dw (rows that end
        // inside 16 bytes would be written past their end)
        const int64_t es = s.f32 ? 4 : 2;
        const bool direct = p->dw_col == 1 && p->dw_row * es % 16 == 0 && D * es % 16 == 0 && p->dw_row >= D &&
                            (reinterpret_cast<uintptr_t>(c.dw) & 15) == 0 && s.rows >= T;
        s.dw = choose_spread(nv, D, n, terms, tallest, true,
                             direct ? float(nv) * float(D) * float(8 + es) / 6.0e6f : 0.0f);
        if (!direct || s.dw.splits > 1) s.dw_sum_rows = sum_rows(nv, D, s.dw.shape);
    }

    Bump measure{nullptr, 0};
    lay_out(measure, c, s);
    void* ws = nullptr;
    int dev = 0;
    SW_CUDA_TRY(cudaGetDevice(&dev), "cudaGetDevice");
    const int pooled = keep_pool_memory(dev);
    if (pooled != SW_OK) return pooled;
    cudaError_t err = cudaMallocAsync(&ws, (size_t)measure.used, stream);
    if (err == cudaErrorMemoryAllocation) {
        cudaGetLastError();
        return fail(SW_ERR_NOMEM, "%s: out of device memory for %lld bytes of workspace", name,
                    (long long)measure.used);
    }
    SW_CUDA_TRY(err, "cudaMallocAsync (linear head workspace)");
    Bump real{static_cast<uint8_t*>(ws), 0};
    const Layout l = lay_out(real, c, s);
    const int rc = s.f32 ? run<true>(c, s, l, stream) : run<false>(c, s, l, stream);
    const cudaError_t freed = cudaFreeAsync(ws, stream);
    if (rc != SW_OK) return rc;
    SW_CUDA_TRY(freed, "cudaFreeAsync (linear head workspace)");
    return ok();
}

}  // namespace
}  // namespace head
}  // namespace sw

extern "C" int sw_linear_xent(const sw_linear_head* plan, const void* h, const void* w, const int32_t* targets,
                              int32_t ignore_index, float logit_scale, float* loss, float* lse, const float* upstream,
                              void* dh, void* dw, void* stream) {
    using namespace sw;
    if (plan && plan->tokens > 0 && !targets) return fail(SW_ERR_INVALID, "sw_linear_xent: null targets");
    static const int32_t none = 0;  // no rows: the list is never read
    head::Call c;
    memset(&c, 0, sizeof(c));
    c.plan = plan;
    c.h = h;
    c.w = w;
    c.targets = targets ? targets : &none;
    c.ignore_index = ignore_index;
    c.top_k = 1;
    c.scale = logit_scale;
    c.factor = 1.0f;
    c.loss = loss;
    c.lse = lse;
    c.upstream = upstream;
    c.dh = dh;
    c.dw = dw;
    return head::check_and_run("sw_linear_xent", c, stream);
}

extern "C" int sw_linear_distill(const sw_linear_head* plan, const void* h, const void* w, const int32_t* index,
                                 const float* logits, int32_t top_k, float temperature, float* loss, float* lse,
                                 const float* upstream, void* dh, void* dw, void* stream) {
    using namespace sw;
    if (plan && plan->tokens > 0 && (!index || !logits))
        return fail(SW_ERR_INVALID, "sw_linear_distill: null teacher entries");
    if (top_k < 1 || top_k > SW_MAX_TEACHER)
        return fail(SW_ERR_INVALID, "sw_linear_distill: 1 to %d teacher entries a row (got %d)", SW_MAX_TEACHER,
                    (int)top_k);
    if (!(temperature > 0.0f) || !std::isfinite(temperature))
        return fail(SW_ERR_INVALID, "sw_linear_distill: the temperature must be positive and finite");
    head::Call c;
    memset(&c, 0, sizeof(c));
    c.plan = plan;
    c.h = h;
    c.w = w;
    c.teacher_index = index;
    c.teacher_logits = logits;
    c.top_k = top_k;
    c.scale = 1.0f / temperature;
    c.factor = temperature * temperature;
    c.loss = loss;
    c.lse = lse;
    c.upstream = upstream;
    c.dh = dh;
    c.dw = dw;
    return head::check_and_run("sw_linear_distill", c, stream);
}
