// sw_head_gemm.cuh - the 16-bit tensor-core contraction behind the linear
// head's losses (sw_linear_head.cu): C = A B^T with fp32 accumulation in TMEM
// (tcgen05.mma kind::f16, both operands bf16 or both f16), either operand
// K-major or MN-major in memory, and an epilogue per use:
//
//   kEpiLse   logits tile -> per row its maximum, the sum of exp2 against it
//             and the target terms: the logits themselves are not stored
//   kEpiGrad  logits tile -> gradient of the loss with respect to the logits,
//             rounded once to the operand type
//   kEpiOut   the product itself: a gradient of the states or of the weights
//
// One persistent CTA per SM walks 128 x BN tiles.  Warp 0 feeds a ring of
// 64-deep K stages by TMA (128-byte swizzle), one thread of warp 1 issues the
// MMAs, warps 2-9 drain one of two TMEM accumulators while the other is being
// filled: warp w reads TMEM sub-partition w % 4 (32 rows) and one half of the
// tile's columns.  Float32 operands come as two f16 planes (hi + lo of a
// power-of-two multiple of the value): the K walk then runs over three plane
// pairs, hi lo + lo hi + hi hi, which keeps 22 bits of each factor.
//
// The tensor core's fp32 accumulator drops the bits below its last place, so a
// long K walk drifts: measured 1.3e-9 per K element, 1.5e-4 over 128000.  Where
// the result is Float32 (kChunked) the walk is cut into kChunkSteps stages, and
// the epilogue adds the pieces in registers, rounded to nearest.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>
#include <math.h>

#include "sw_common.cuh"
#include "sw_ptx.cuh"

namespace sw {
namespace head {

constexpr int kBM = 128;
constexpr int kBK = 64;                 // K elements of a stage: one 128-byte swizzle row
constexpr int kChunkSteps = 8;          // K stages between two register sums (512 elements of K)
constexpr int kEntryTile = 256;         // columns per entry of the target offset table
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

enum { kEpiLse = 0, kEpiGrad = 1, kEpiOut = 2 };
enum { kCountNone = 0, kCountM = 1, kCountK = 2 };

// What the preparation kernels leave for the contractions.
struct HeadState {
    int count;               // rows that count (compact rows)
    int bad;                 // a target outside the vocabulary was seen
    uint32_t amax[3];        // largest finite |h|, |w|, |row factor| as float bits (Float32 only)
    float grad_scale;        // common factor of every row's gradient, applied to dh and dw in fp32
    int pad[2];
};

// Power-of-two multiplier that brings values of magnitude `amax` just under
// 2^15 (f16 holds up to 65504): exponent q, so that x 2^q is the value split.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
    if (amax_bits == 0) return 0;
    const int e = int(amax_bits >> 23) - 127;
    return min(14 - e, 126);
}
__device__ __forceinline__ float pow2i(int q) { return __uint_as_float(uint32_t(q + 127) << 23); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Placement of an operand's 64-element blocks and of its lo plane, in TMA
// coordinates: block b of plane p starts at element b x_block + p x_plane of a
// row, row r at row r + p y_plane.
struct Plane {
    int x_block, x_plane, y_plane;
};

struct GemmArgs {
    int M, N, K;
    int count_is;            // which extent the device-side row count bounds
    const HeadState* state;
    int row0;                // first compact row of this launch (the count starts there)
    int terms;               // plane pairs walked: 1, or 3 for Float32
    Plane pa, pb;            // where each operand's lo plane and 64-element blocks lie
    int splits;              // parts of the K walk, each with its own slot of `accum`
    int scale_a, scale_b;    // indexes into HeadState::amax of the operands' scales (-1: none)
    // logits epilogues
    float logit_scale;
    int64_t v0;              // first vocabulary column of this piece
    const int* ent_idx;      // [rows][ent_k] target columns, ascending
    const float* ent_p;      // their probabilities (null: 1)
    const uint16_t* offs;    // [tile][rows_pad] first entry of each kEntryTile columns (null: one entry a row)
    int ent_k;
    int rows_pad;
    float4* partial;         // kEpiLse: [half tile][rows_pad] (max, sum, target term, -) in base-2 units
    float* ent_s;            // kEpiLse: base-2 logit of every target entry (null: not kept)
    int keep;                // kEpiLse: write exp2(logit - half tile's max) where the logits' gradient will be
    const float* lse2;       // kEpiGrad: per compact row
    const float* coef;
    uint16_t* grad;          // [rows_pad][ld_grad]; Float32: every 64 columns as 64 hi then 64 lo values
    int64_t ld_grad;         // 16-bit elements
    // kEpiOut
    float* accum;            // fp32 running sums [splits][M][ld_accum] (null: none)
    int64_t ld_accum, slot;
    int first, last;         // first: nothing to add yet; last: write dst
    void* dst;
    int dst_f32;
    int64_t dst_row, dst_col;
    const int* row_map;      // destination row of each row (null: itself)
};

template <int BN, int kStages>
struct Cfg {
    static constexpr int kThreads = 64 + 256;
    static constexpr int kABytes = kBM * kBK * 2;
    static constexpr int kBBytes = BN * kBK * 2;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kOffBar = kStages * kStageBytes;
    static constexpr int kNumBars = 2 * kStages + 5;
    static constexpr int kOffSlot = kOffBar + kNumBars * 8;
    static constexpr int kSmemBytes = kOffSlot + 16 + 1024;
    static constexpr int kTmemCols = 2 * BN;
    static_assert(kSmemBytes <= 232448, "shared memory budget");
};

// D[tmem] (+)= A[smem] B[smem], 16-bit operands, fp32 accumulation.
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Instruction descriptor of kind::f16: fp32 D; both operands bf16 or both f16;
// a major bit of 1 marks an MN-major operand.
__device__ __forceinline__ uint32_t idesc_f16(bool bf16, bool a_mn, bool b_mn, int M, int N) {
    const uint32_t fmt = bf16 ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
           (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

// Loads 16 consecutive 32-bit TMEM columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// The target entries of one row inside a tile: a cursor over its ascending
// list.  Rows are spread over a warp's lanes, and `take` runs for every entry
// inside the 32 columns that the warp holds in registers.
struct EntryCursor {
    const int* idx;
    const float* p;
    int e, end;
    int next;  // column of entry e, INT_MAX past the end

    __device__ __forceinline__ void load() { next = e < end ? idx[e] : INT_MAX; }
    __device__ __forceinline__ void begin(const GemmArgs& a, int64_t row, bool row_in, int64_t col0) {
        e = 0;
        end = 0;
        idx = a.ent_idx + row * a.ent_k;
        p = a.ent_p ? a.ent_p + row * a.ent_k : nullptr;
        if (row_in) {
            if (a.offs) {
                const int64_t tile = col0 / kEntryTile;
                e = a.offs[tile * a.rows_pad + row];
                end = a.offs[(tile + 1) * a.rows_pad + row];
            } else {
                end = 1;
            }
        }
        load();
        while (next < col0) {
            ++e;
            load();
        }
    }
    template <class F>
    __device__ __forceinline__ void walk(int64_t chunk0, F&& take) {
        int64_t rel = int64_t(next) - chunk0;
        while (__any_sync(0xffffffffu, rel < 32)) {
            const bool mine = rel < 32;
            take(mine ? int(rel) : -1, mine ? (p ? p[e] : 1.0f) : 0.0f);
            if (mine) {
                ++e;
                load();
                rel = int64_t(next) - chunk0;
            }
        }
    }
};

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (kBf16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&v);
    }
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}

template <bool kBf16>
__device__ __forceinline__ void store_row32(uint16_t* dst, const float (&r)[32]) {
    uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
    for (int v = 0; v < 4; ++v)
        d[v] = make_uint4(pack2<kBf16>(r[8 * v], r[8 * v + 1]), pack2<kBf16>(r[8 * v + 2], r[8 * v + 3]),
                          pack2<kBf16>(r[8 * v + 4], r[8 * v + 5]), pack2<kBf16>(r[8 * v + 6], r[8 * v + 7]));
}

// Where 32 columns of a row's logits' gradient are: column n0 of the row, and
// in Float32 its hi values (the lo values 64 elements further).
template <bool kBf16>
__device__ __forceinline__ uint16_t* grad_at(const GemmArgs& args, int64_t m, int64_t n0) {
    return args.grad + m * args.ld_grad + (kBf16 ? n0 : (n0 & ~int64_t(63)) * 2 + (n0 & 63));
}

// Softmax statistics of a row over the half tile in registers, in base-2
// units: ref = max k2 z, sum of exp2(k2 z - ref), target term sum p z.  With
// `keep` the exponentials are stored too, for the gradient: as f16 times 2^15
// (11 bits down to 2^-29 of the half tile's largest; the later rounding to
// bf16 is the one that counts) or, for Float32, as they are.
template <bool kBf16, int kParts>
__device__ __forceinline__ float4 lse_tile(const GemmArgs& args, EntryCursor& cur, int64_t m, int64_t n0, bool row_in,
                                           float k2, float (&r)[kParts][32]) {
    float dot = 0.0f, top = -INFINITY;
#pragma unroll
    for (int c = 0; c < kParts; ++c) {
        cur.walk(args.v0 + n0 + c * 32, [&](int rel, float p) {
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j == rel) v = r[c][j];
            if (rel >= 0) {
                dot += p * v;
                if (args.ent_s) args.ent_s[m * args.ent_k + cur.e] = v * k2;
            }
        });
        const int ncols = (int)min(int64_t(32), int64_t(args.N) - (n0 + c * 32));
        if (ncols < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j >= ncols) r[c][j] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) top = fmaxf(top, r[c][j]);
    }
    const float ref = top * k2;
    // columns of nothing but -inf add nothing (and must not make -inf minus -inf)
    const float base = ref == -INFINITY ? 0.0f : ref;
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < kParts; ++c) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            r[c][j] = ex2(fmaf(r[c][j], k2, -base));
            sum += r[c][j];
        }
        // (Float32 blocks of 64 columns are written whole: the K walk reads them whole)
        if (args.keep && n0 + c * 32 < (kBf16 ? int64_t(args.N) : (int64_t(args.N) + 63) / 64 * 64)) {
            if (kBf16) {
#pragma unroll
                for (int j = 0; j < 32; ++j) r[c][j] = row_in ? r[c][j] * 32768.0f : 0.0f;
                store_row32<false>(grad_at<true>(args, m, n0 + c * 32), r[c]);
            } else {
                float4* d = reinterpret_cast<float4*>(args.grad + m * args.ld_grad + 2 * (n0 + c * 32));
#pragma unroll
                for (int v = 0; v < 8; ++v)
                    d[v] = row_in ? make_float4(r[c][4 * v], r[c][4 * v + 1], r[c][4 * v + 2], r[c][4 * v + 3])
                                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
    }
    return make_float4(ref, sum, dot * k2, 0.0f);
}

// Gradient with respect to 32 logits of a row: softmax minus target in fp32,
// rounded once to the type the next contractions read.  Float32: zeros up to
// the end of a 64-column block, which the K walk reads whole.
template <bool kBf16>
__device__ __forceinline__ void grad_part(const GemmArgs& args, EntryCursor& cur, int64_t m, int64_t n0, int ncols,
                                          bool row_in, float k2, float lse2, float coef, float (&r)[32]) {
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] = ex2(fmaf(r[j], k2, -lse2));
    cur.walk(args.v0 + n0, [&](int rel, float p) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j == rel) r[j] -= p;
    });
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] = row_in && j < ncols ? r[j] * coef : 0.0f;
    uint16_t* d = grad_at<kBf16>(args, m, n0);
    store_row32<kBf16>(d, r);
    if (!kBf16) {
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] -= __half2float(__float2half_rn(r[j]));
        store_row32<kBf16>(d + 64, r);
    }
}

// 32 columns of a result row: scaled, added to the running fp32 sum, and the
// last time written in the result's type.
__device__ __forceinline__ void out_part(const GemmArgs& args, int split, int64_t m, int64_t n0, int ncols,
                                         float scale, float (&r)[32]) {
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] *= scale;
    if (args.accum) {
        float* a = args.accum + split * args.slot + m * args.ld_accum + n0;
        const bool whole = ncols == 32 && (reinterpret_cast<uintptr_t>(a) & 15) == 0;
        if (!args.first) {
            if (whole) {
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    const float4 o = reinterpret_cast<const float4*>(a)[v];
                    r[4 * v] += o.x;
                    r[4 * v + 1] += o.y;
                    r[4 * v + 2] += o.z;
                    r[4 * v + 3] += o.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (j < ncols) r[j] += a[j];
            }
        }
        if (!args.last) {
            if (whole) {
#pragma unroll
                for (int v = 0; v < 8; ++v)
                    reinterpret_cast<float4*>(a)[v] = make_float4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (j < ncols) a[j] = r[j];
            }
            return;
        }
    }
    const int64_t row = args.row_map ? args.row_map[m] : m;
    if (args.dst_f32) {
        float* d = static_cast<float*>(args.dst) + row * args.dst_row + n0 * args.dst_col;
        if (ncols == 32 && args.dst_col == 1 && (reinterpret_cast<uintptr_t>(d) & 15) == 0) {
#pragma unroll
            for (int v = 0; v < 8; ++v)
                reinterpret_cast<float4*>(d)[v] = make_float4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j < ncols) d[j * args.dst_col] = r[j];
        }
    } else {
        __nv_bfloat16* d = static_cast<__nv_bfloat16*>(args.dst) + row * args.dst_row + n0 * args.dst_col;
        if (ncols == 32 && args.dst_col == 1 && (reinterpret_cast<uintptr_t>(d) & 15) == 0) {
            store_row32<true>(reinterpret_cast<uint16_t*>(d), r);
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j < ncols) d[j * args.dst_col] = __float2bfloat16_rn(r[j]);
        }
    }
}

template <int BN, int kStages, bool kBf16, bool kAMn, bool kBMn, int kEpi, bool kChunked>
__global__ void __launch_bounds__(320, 1)
    head_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                     const GemmArgs args) {
    using C = Cfg<BN, kStages>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = ptx::smem_addr(smem);
    const uint32_t bar_full = sbase + C::kOffBar;
    const uint32_t bar_empty = bar_full + kStages * 8;
    const uint32_t bar_tmem_full = bar_empty + kStages * 8;  // two accumulators
    const uint32_t bar_tmem_empty = bar_tmem_full + 16;
    const uint32_t bar_drain = bar_tmem_empty + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffSlot);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(bar_full + 8 * s, 1);
            ptx::mbar_init(bar_empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            ptx::mbar_init(bar_tmem_full + 8 * b, 1);
            ptx::mbar_init(bar_tmem_empty + 8 * b, 256);
        }
        ptx::mbar_init(bar_drain, 1);
        ptx::fence_barrier_init();
        ptx::prefetch_tmap(&tmap_a);
        ptx::prefetch_tmap(&tmap_b);
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_addr(tmem_slot), C::kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_enter();

    const int count = args.count_is == kCountNone ? 0 : max(args.state->count - args.row0, 0);
    const int M = args.count_is == kCountM ? min(args.M, count) : args.M;
    const int K = args.count_is == kCountK ? min(args.K, count) : args.K;
    const int num_m = (M + kBM - 1) / kBM;
    const int num_n = (args.N + BN - 1) / BN;
    const int num_tiles = num_m * num_n;
    const int num_items = num_tiles * args.splits;
    const int k_steps = (K + kBK - 1) / kBK;
    const int split_steps = (k_steps + args.splits - 1) / args.splits;
    constexpr int kGroup = 16;
    // Work item `t`: a tile and its share [k0, k1) of the K stages.
    auto item = [&](int t, int& mb, int& nb, int& split, int& k0, int& k1) {
        split = t / num_tiles;
        t -= split * num_tiles;
        k0 = min(split * split_steps, k_steps);
        k1 = min(k0 + split_steps, k_steps);
        const int per_group = kGroup * num_n;
        const int g = t / per_group;
        const int first = g * kGroup;
        const int gsize = min(num_m - first, kGroup);
        const int r = t % per_group;
        mb = first + r % gsize;
        nb = r / gsize;
    };
    auto chunk_end = [&](int k0, int k1) { return kChunked ? min(k0 + kChunkSteps, k1) : k1; };

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            uint32_t issued[kStages] = {0};
            bool alive = true;
            for (int t = blockIdx.x; t < num_items && alive; t += gridDim.x) {
                int mb, nb, split, k0, k1;
                item(t, mb, nb, split, k0, k1);
                for (int c0 = k0; c0 < k1 && alive; c0 = chunk_end(c0, k1))
                    for (int term = 0; term < args.terms && alive; ++term) {
                        // plane pairs, the small products first: (hi, lo), (lo, hi), (hi, hi)
                        const int pa = args.terms == 3 && term == 1;
                        const int pb = args.terms == 3 && term == 0;
                        const int xa = pa * args.pa.x_plane, ya = pa * args.pa.y_plane;
                        const int xb = pb * args.pb.x_plane, yb = pb * args.pb.y_plane;
                        const int c1 = chunk_end(c0, k1);
                        for (int ks = c0; ks < c1; ++ks) {
                            if (!ptx::mbar_wait(bar_empty + 8 * stage, phase ^ 1)) { alive = false; break; }
                            const uint32_t full = bar_full + 8 * stage;
                            const uint32_t sa = sbase + stage * C::kStageBytes;
                            const uint32_t sb = sa + C::kABytes;
                            ptx::mbar_arrive_expect_tx(full, C::kStageBytes);
                            if (kAMn) {
#pragma unroll
                                for (int g = 0; g < kBM / 64; ++g)
                                    ptx::tma_load_2d(sa + g * 8192, &tmap_a,
                                                     (mb * (kBM / 64) + g) * args.pa.x_block + xa, ya + ks * kBK, full);
                            } else {
                                ptx::tma_load_2d(sa, &tmap_a, ks * args.pa.x_block + xa, ya + mb * kBM, full);
                            }
                            if (kBMn) {
#pragma unroll
                                for (int g = 0; g < BN / 64; ++g)
                                    ptx::tma_load_2d(sb + g * 8192, &tmap_b,
                                                     (nb * (BN / 64) + g) * args.pb.x_block + xb, yb + ks * kBK, full);
                            } else {
                                ptx::tma_load_2d(sb, &tmap_b, ks * args.pb.x_block + xb, yb + nb * BN, full);
                            }
                            issued[stage] += 1;
                            if (++stage == kStages) { stage = 0; phase ^= 1; }
                        }
                    }
            }
            for (int s = 0; s < kStages; ++s)
                if (issued[s] > 0) ptx::mbar_wait(bar_full + 8 * s, (issued[s] - 1) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = idesc_f16(kBf16, kAMn, kBMn, kBM, BN);
            int stage = 0;
            uint32_t phase = 0, it = 0;
            bool alive = true;
            for (int t = blockIdx.x; t < num_items && alive; t += gridDim.x) {
                int mb, nb, split, k0, k1;
                item(t, mb, nb, split, k0, k1);
                for (int c0 = k0; c0 < k1; c0 = chunk_end(c0, k1), ++it) {
                    const uint32_t buf = it & 1;
                    if (!ptx::mbar_wait(bar_tmem_empty + 8 * buf, ((it >> 1) & 1) ^ 1)) { alive = false; break; }
                    ptx::tc_fence_after();
                    const uint32_t acc = tmem + buf * BN;
                    const int steps = (chunk_end(c0, k1) - c0) * args.terms;
                    for (int ks = 0; ks < steps; ++ks) {
                        if (!ptx::mbar_wait(bar_full + 8 * stage, phase)) { alive = false; break; }
                        ptx::tc_fence_after();
                        const uint32_t sa = sbase + stage * C::kStageBytes;
                        const uint32_t sb = sa + C::kABytes;
#pragma unroll
                        for (int j = 0; j < kBK / 16; ++j) {
                            // K-major: 16 elements of K are 32 bytes of the swizzled row, 8-row groups 1024
                            // bytes apart.  MN-major: 16 rows of K are 2048 bytes, 64-element blocks of the
                            // other mode 8192 bytes apart, 8-row groups of K 1024.
                            const uint64_t ad = kAMn ? ptx::smem_desc(sa + 2048 * j, 8192, 1024, ptx::kLayoutSwizzle128)
                                                     : ptx::smem_desc(sa + 32 * j, 0, 1024, ptx::kLayoutSwizzle128);
                            const uint64_t bd = kBMn ? ptx::smem_desc(sb + 2048 * j, 8192, 1024, ptx::kLayoutSwizzle128)
                                                     : ptx::smem_desc(sb + 32 * j, 0, 1024, ptx::kLayoutSwizzle128);
                            mma_f16(acc, ad, bd, idesc, (ks > 0 || j > 0) ? 1u : 0u);
                        }
                        ptx::tc_commit(bar_empty + 8 * stage);
                        if (++stage == kStages) { stage = 0; phase ^= 1; }
                    }
                    if (!alive) break;
                    ptx::tc_commit(bar_tmem_full + 8 * buf);
                }
            }
            ptx::tc_commit(bar_drain);
            ptx::mbar_wait(bar_drain, 0);
        }
    } else {
        constexpr int kCols = BN / 2;     // columns of this warp: half of the tile
        constexpr int kParts = kCols / 32;
        const int quarter = warp & 3;
        const int half = (warp - 2) >> 2;
        const int row_in_tile = quarter * 32 + lane;
        // inverse of the operands' power-of-two scales
        float inv = 1.0f;
        if (args.scale_a >= 0) inv *= pow2i(-scale_exponent(args.state->amax[args.scale_a]));
        if (args.scale_b >= 0) inv *= pow2i(-scale_exponent(args.state->amax[args.scale_b]));
        const float k2 = args.logit_scale * kLog2e * inv;
        const float gscale = kEpi == kEpiGrad && !kBf16 ? pow2i(scale_exponent(args.state->amax[2])) : 1.0f;
        const float out_scale = kEpi == kEpiOut ? inv * args.state->grad_scale : 1.0f;
        uint32_t it = 0;
        bool alive = true;
        for (int t = blockIdx.x; t < num_items && alive; t += gridDim.x) {
            int mb, nb, split, k0, k1;
            item(t, mb, nb, split, k0, k1);
            const int64_t m = int64_t(mb) * kBM + row_in_tile;
            const bool row_in = m < M;
            const int64_t ncol0 = int64_t(nb) * BN + half * kCols;
            EntryCursor cur;
            float lse2 = 0.0f, coef = 0.0f;
            if (kEpi != kEpiOut) cur.begin(args, m, row_in, args.v0 + ncol0);
            if (kEpi == kEpiGrad && row_in) {
                lse2 = args.lse2[m];
                coef = args.coef[m] * gscale;
            }
            // one 32-column part of the finished accumulator
            auto part = [&](int c, float (&r)[32]) {
                const int64_t n0 = ncol0 + c * 32;
                const int ncols = (int)max(int64_t(0), min(int64_t(32), int64_t(args.N) - n0));
                if (kEpi == kEpiGrad) {
                    if (n0 < (int64_t(args.N) + 63) / 64 * 64)
                        grad_part<kBf16>(args, cur, m, n0, ncols, row_in, k2, lse2, coef, r);
                } else if (kEpi == kEpiOut) {
                    if (row_in && ncols) out_part(args, split, m, n0, ncols, out_scale, r);
                }
            };
            if (kChunked) {
                float sum[kParts][32];
#pragma unroll
                for (int c = 0; c < kParts; ++c)
#pragma unroll
                    for (int j = 0; j < 32; ++j) sum[c][j] = 0.0f;
                for (int c0 = k0; c0 < k1; c0 = chunk_end(c0, k1), ++it) {
                    const uint32_t buf = it & 1;
                    if (!ptx::mbar_wait(bar_tmem_full + 8 * buf, (it >> 1) & 1)) { alive = false; break; }
                    __syncwarp();
                    ptx::tc_fence_after();
                    const uint32_t acc = tmem + buf * BN + half * kCols + (uint32_t(quarter * 32) << 16);
#pragma unroll
                    for (int c = 0; c < 2 * kParts; ++c) {
                        uint32_t u[16];
                        tmem_ld_32x32b_x16(acc + c * 16, u);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) sum[c / 2][c % 2 * 16 + j] += __uint_as_float(u[j]);
                    }
                    ptx::tc_fence_before();
                    ptx::mbar_arrive(bar_tmem_empty + 8 * buf);
                }
                if (!alive) break;
                if (kEpi == kEpiLse) {
                    const float4 st = lse_tile<kBf16, kParts>(args, cur, m, ncol0, row_in, k2, sum);
                    args.partial[(args.v0 + ncol0) / kCols * args.rows_pad + m] = st;
                } else {
#pragma unroll
                    for (int c = 0; c < kParts; ++c) part(c, sum[c]);
                }
            } else {
                const uint32_t buf = it & 1;
                const bool any = k0 < k1;  // an empty share has no accumulator: zeros
                if (any) {
                    if (!ptx::mbar_wait(bar_tmem_full + 8 * buf, (it >> 1) & 1)) break;
                    ptx::tc_fence_after();
                }
                const uint32_t acc = tmem + buf * BN + half * kCols + (uint32_t(quarter * 32) << 16);
#pragma unroll 1
                for (int c = 0; c < kParts; ++c) {
                    __syncwarp();
                    uint32_t u[32];
                    float r[32];
                    ptx::tmem_ld_32x32b_x32(acc + c * 32, u);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = any ? __uint_as_float(u[j]) : 0.0f;
                    part(c, r);
                }
                if (any) {
                    ptx::tc_fence_before();
                    ptx::mbar_arrive(bar_tmem_empty + 8 * buf);
                    ++it;
                }
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    if (warp == 1) ptx::tmem_dealloc(tmem, C::kTmemCols);
}

}  // namespace head
}  // namespace sw
