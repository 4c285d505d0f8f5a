// sw_head_gemm.cuh - the 16-bit tensor-core contraction behind the linear
// head's losses (sw_linear_head.cu): C = A B^T with fp32 accumulation in TMEM
// (tcgen05.mma kind::f16, both operands bf16 or both f16), either operand
// K-major or MN-major in memory, and an epilogue per use:
//
//   kEpiLse   logits tile -> per row its maximum, the sum of exp2 against it
//             and the target terms: the logits themselves are not stored
//   kEpiGrad  logits tile -> gradient of the loss with respect to the logits,
//             rounded once to the operand type
//   kEpiGradCut  the same in bf16 where the K walk is cut into pieces (below): the
//             registers of that cost 4 % of a call whose walk is one piece, dim 1024
//   kEpiOut   the product itself: a gradient of the states or of the weights
//
// Tile shapes (kShape), on persistent CTAs:
//   kSingle  128 x 256 on one CTA;
//   kPair2   256 x 256 on a pair of CTAs on neighbouring SMs, tcgen05
//            cta_group::2: each CTA holds its 128 rows of A and half of B in
//            shared memory and its rows of the accumulator in TMEM, so a K
//            stage moves 32 KiB per SM instead of 48;
//   kTall    512 x 256 on a pair: two accumulators of 256 x 256 that share B, a
//            stage of 48 KiB per SM for twice the work.  Nothing is left of TMEM
//            for a second tile, so about 3000 cycles of a tile's epilogue are not
//            hidden; in exchange a quarter fewer bytes come from L2, which under
//            the power limit buys clock.
// Warp 0 feeds a ring of 64-deep K stages by TMA (128-byte swizzle), one elected
// lane of warp 1 (of the pair's first CTA) issues the MMAs (from a warp that
// stays in step: a lone thread took about 350 cycles for a stage's four MMAs, of
// the 512 that they last; so it takes 200), warps 2-9 drain one of two TMEM
// accumulators while the other is being filled: warp w reads TMEM
// sub-partition w % 4 (32 rows) and one half of the tile's columns.  Results
// pass through 4 KiB of shared memory per warp, so that they leave as whole
// 128-byte row segments.  Float32 operands come as two f16 planes (hi + lo of a
// power-of-two multiple of the value, one for a whole matrix): the K walk then runs
// over three plane pairs, hi lo + lo hi + hi hi, which keeps 22 bits of each factor
// down to 2^-18 of the matrix's largest, and 2^-40 of that below.  Where a row is
// so far below the others that this would show in it (HeadState::wide), the planes
// are bf16 instead, which have Float32's range: three of an operand (24 bits) and
// two of the logits' gradient (16), multiplied pair by pair down to 2^-16 of the
// largest product.
//
// The tensor core's fp32 accumulator drops the bits below its last place, so a
// long K walk drifts: measured 1.3e-9 per K element, 1.5e-4 over 128000.  Where
// the result is Float32 (kChunked: logits, and Float32 gradients) the walk is cut
// into pieces of args.chunk stages, and the epilogue adds them in registers, rounded
// to nearest.  Logits computed again for their gradient are cut as they were for
// their lse: what both drift by cancels in exp(s - lse), where at s = 60 the drift
// of one alone, 1e-4 over a dim of 2048, would be more than a row sure of its
// target has left.
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
constexpr int kBN = 256;
constexpr int kEntryTile = 256;         // columns per entry of the target offset table
// With at most this many rows that count, one bf16 rounding of a dominant entry
// of the logits' gradient would show in a result (nothing averages it out), and
// three quarters of a tile's rows are idle: rows 64 .. 127 then hold what the
// rounding of rows 0 .. 63 left, against the same states.
constexpr int kFewRows = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLargeExponent = 1048576.0f;  // from here on the rounding of an exponent may be 1/16 and more

enum { kEpiLse = 0, kEpiGrad = 1, kEpiOut = 2, kEpiGradCut = 3 };
enum { kCountM, kCountK };
enum { kKMajor, kMnMajor, kBoth };       // A in memory; kBoth: of two contractions, each its own

// How the tiles of a contraction are walked: groups of row tiles (which share
// B's panels in L2), column tiles inside, row tiles innermost; the workers take
// whole waves of tiles, and the tiles of the last, partial wave are cut into
// `parts` shares of the K walk, each with its own rows of the fp32 sums: part 0
// at the row itself, part p > 0 of rows from `row_f` on behind all rows.
// Groups of 2048 rows: 512 / 1024 / 2048 / 4096 / 8192, an 8192 x 131072 x 4096
// step under the power cap: 25.3 / 25.4 / 24.5 / 24.3 / 25.9 ms, 4096 x 32000 x
// 4096: 2.94 / 2.88 / 2.81 / 2.82 / 2.91.
struct Walk {
    int num_m, num_n, tile_m, group, parts, whole, row_f;

    __host__ __device__ Walk(int M, int cols_tiles, int rows_per_tile, int workers, int parts_)
        : num_m((M + rows_per_tile - 1) / rows_per_tile), num_n(cols_tiles), tile_m(rows_per_tile),
          group(2048 / rows_per_tile), parts(parts_) {
        const int tiles = num_m * num_n;
        whole = parts > 1 ? tiles / workers * workers : tiles;
        row_f = whole / (group * num_n) * group * tile_m;
    }
    __host__ __device__ int items() const { return whole + (num_m * num_n - whole) * parts; }
    __host__ __device__ int tile_of(int mb, int nb) const {
        const int first = mb / group * group;
        return first * num_n + nb * min_(num_m - first, group) + (mb - first);
    }
    __host__ __device__ void coords(int tile, int& mb, int& nb) const {
        const int per_group = group * num_n, first = tile / per_group * group;
        const int rows = min_(num_m - first, group), r = tile - first * num_n;
        nb = r / rows;
        mb = first + r - nb * rows;
    }
    // Row of the sums that holds row m of part p.
    __host__ __device__ int sum_row(int p, int m) const {
        return p == 0 ? m : num_m * tile_m + (p - 1) * (num_m * tile_m - row_f) + (m - row_f);
    }
    __host__ __device__ static int min_(int a, int b) { return a < b ? a : b; }
};

// What the preparation kernel leaves for the others.
struct HeadState {
    int count;               // rows that count (compact rows)
    int bad;                 // a target outside the vocabulary was seen
    // Float32 only, as float bits: largest finite |h|, |w|, |row factor|, and the least
    // of a row that is not zero
    uint32_t amax[3], least[3];
    int wide;                // rows too far apart for f16 planes (from the first split on)
    float grad_scale;        // common factor of every row's gradient, applied to dh and dw in fp32
    int dh_splits;           // parts of the K walk of dh, chosen for the rows that count
    int done;                // rows whose loss is written

    // Rows that count from row0 on, and whether they have remainder rows (bf16).
    __device__ __forceinline__ int rows(int row0) const { return max(count - row0, 0); }
    __device__ __forceinline__ bool few(int row0) const { return count <= kFewRows && rows(row0) > 0; }
};

// Rows this many powers of two below the largest keep 22 bits and more of their
// own largest element in f16 planes (2^-40 of the matrix's largest).  A row's
// gradient with a factor that far below is a sum over the vocabulary of entries
// that are 2^12 coarser: 2^-28 sqrt(131072) = 2^-19 of it.  bf16 planes cost 2008 us
// for 1325 (a step of 2048 x 32000, dim 1024), so they are only for what needs them.
constexpr int kSpread = 16, kFactorSpread = 12;
__device__ __forceinline__ bool rows_far_apart(const HeadState* s) {
    bool far = false;
    for (int q = 0; q < 3; ++q) {
        const uint32_t most = s->amax[q], least = s->least[q];
        far |= least < most && int(most >> 23) - int(least >> 23) > (q == 2 ? kFactorSpread : kSpread);
    }
    return far;
}

// Power-of-two multiplier that brings values of magnitude `amax` just under
// 2^15 (f16 holds up to 65504; bf16 planes are for small rows, which 2^23 keeps
// from the subnormals): exponent q, so that x 2^q is the value split.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits, bool wide) {
    if (amax_bits == 0) return 0;
    const int e = int(amax_bits >> 23) - 127;
    return min((wide ? 22 : 14) - e, 126);
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

// One contraction of a launch.
struct Problem {
    int M, N, K;
    int count_is;            // which extent the device-side row count bounds
    int a_mn;                // A is MN-major in memory (gradients of the weights)
    Plane pa, pb;            // where each operand's lo plane and 64-element blocks lie
    int splits;              // parts of the last wave's tiles (0: state->dh_splits)
    int scale_a, scale_b;    // indexes into HeadState::amax of the operands' scales (-1: none)
    // kEpiOut, through the output map: the result in its type, or fp32 running
    // sums, with rows as Walk places them
    int sums;
    int first;               // nothing to add yet
};

// Tensor maps of the operands and of what is written, per contraction.
struct alignas(64) Maps {
    CUtensorMap a[2], b[2], c[2];
};

// Plane of an operand in product `term` of the planes' products, the smallest
// first (lists of hexadecimal digits, the first product's last): bf16 values have
// one plane; f16 planes (0, 1), (1, 0), (0, 0); bf16 planes of Float32 the six, or
// with a gradient's two planes five, whose numbers add up to 2 at most.
struct Products {
    int terms;
    uint32_t a, b;
};
__device__ __forceinline__ Products products(bool f32, bool wide, bool gradient) {
    if (!f32) return Products{1, 0, 0};
    if (!wide) return Products{3, 0x010, 0x001};
    return gradient ? Products{5, 0x01010, 0x00112} : Products{6, 0x010210, 0x001012};
}
__device__ __forceinline__ int plane_of(uint32_t list, int term) { return list >> (4 * term) & 15; }

struct GemmArgs {
    Problem p[2];            // two at once: the gradients of states and weights of few rows
    int problems;
    int alternate;           // every second worker takes the second one first
    const HeadState* state;
    int row0;                // first compact row of this launch (the count starts there)
    int terms;               // plane pairs walked, for estimates: 1, or 3 for Float32
    int chunk;               // K stages between two sums in registers (kChunked)
    // logits epilogues
    float logit_scale;
    int64_t v0;              // first vocabulary column of this piece
    const int* ent_idx;      // [rows][ent_k] target columns, ascending
    const float* ent_p;      // their probabilities (null: 1)
    const uint16_t* offs;    // [tile][rows_pad] first entry of each kEntryTile columns (null: one entry a row)
    int ent_k;
    int rows_pad;
    float4* partial;         // kEpiLse: [rows][slots] (max, sum, target term, unused: one store)
    int slots, slot_shift;   // a slot for each 1 << slot_shift columns: 128, or a narrow tile's 64
    int tile_n;              // logits tiles of one CTA: 256 columns, or 128 or 64 where they spread over more SMs
    float* ent_s;            // kEpiLse: h w of every target entry (null: not kept)
    int keep;                // kEpiLse: write exp2(logit - half tile's max) where the logits' gradient will be
    // kEpiGrad: softmax(z) = exp2((z to_ref - norm.x) to_log2 - norm.y), norm per compact
    // row; exp2's factor of z is logit_scale log2(e) rounded, and to_ref to_log2 less
    // that, over to_ref, is factor_rest
    const float2* norm;
    float to_ref, to_log2, factor_rest;
    const float* coef;
};

enum { kSingle = 0, kPair2 = 1, kTall = 2 };
__host__ __device__ constexpr int shape_rows(int shape) { return kBM << shape; }

template <int kShape>
struct Cfg {
    static constexpr bool kPair = kShape != kSingle;
    static constexpr int kAccs = kShape == kTall ? 2 : 1;  // accumulators of one tile
    static constexpr int kThreads = 64 + 256;
    static constexpr int kTileM = shape_rows(kShape);
    static constexpr int kAccRows = kPair ? 2 * kBM : kBM; // rows of one accumulator over the CTAs
    static constexpr int kBRows = kPair ? kBN / 2 : kBN;  // rows of B that one CTA holds
    static constexpr int kABytes = kAccs * kBM * kBK * 2;
    static constexpr int kBBytes = kBRows * kBK * 2;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kStages = kShape == kPair2 ? 5 : 4;
    static constexpr int kBoxes = kShape == kPair2 ? 2 : 1;           // 4 KiB staging boxes per epilogue warp
    static constexpr int kOffOut = kStages * kStageBytes;
    static constexpr int kOffBar = kOffOut + 8 * kBoxes * 4096;
    static constexpr int kNumBars = 2 * kStages + 5;
    static constexpr int kOffSlot = kOffBar + kNumBars * 8;
    static constexpr int kSmemBytes = kOffSlot + 16 + 1024;
    static constexpr int kTmemCols = 2 * kBN;
    static_assert(kSmemBytes <= 232448, "shared memory budget");
};

// Estimated microseconds of a K stage, and of a tile's fill and drain that
// nothing hides: a stage takes 0.26 us on a pair (256 x 256) or 0.52 (tall), and on a
// single CTA, half the work, 0.32 where all SMs draw their 48 KiB a stage from L2 (0.27
// on a few; at 0.27 a step of 1024 x 32000 at dim 2048 takes single tiles for dw
// and 413 us, at 0.32 pairs and 390).
__host__ __device__ inline float stage_us(int shape, int terms) {
    return float(terms) * (shape == kTall ? 0.52f : shape == kPair2 ? 0.26f : 0.32f);
}
__host__ __device__ inline float fixed_us(int shape) { return shape == kTall ? 5.0f : shape == kPair2 ? 2.5f : 2.0f; }
__host__ __device__ inline int shape_workers(int shape, int sms) { return shape == kSingle ? sms : sms / 2; }

// A contraction of a launch as one worker sees it: its tiles and K stages, and
// which work items are its own, item i: `pre` of them come before the workers'
// common rounds (see below).
struct Plan {
    Walk walk;
    int items, k_steps, part_steps;
    int pre, pre_first, pre_stride, pool;

    __device__ __forceinline__ Plan(int M, int N, int K, int tile_m, int tile_n, int workers, int parts)
        : walk(M, (N + tile_n - 1) / tile_n, tile_m, workers, parts), items(walk.items()), k_steps((K + kBK - 1) / kBK),
          part_steps((k_steps + parts - 1) / parts), pre(0), pre_first(0), pre_stride(0), pool(0) {}
    // The contraction `before` left all workers but the first items % workers
    // one item ahead: they take `gain` items of this one first, as many as last
    // as long as one of the other's.
    __device__ __forceinline__ void follow(const Plan& before, int worker, int workers, float stage, float fixed) {
        const int rest = before.items % workers;
        if (rest == 0) return;
        const int gain = int((float(before.part_steps) * stage + fixed) / (float(part_steps) * stage + fixed) + 0.5f);
        pre_stride = workers - rest;
        pool = int(min(int64_t(items), int64_t(pre_stride) * gain));
        pre_first = worker - rest;
        if (pre_first >= 0 && pre_first < pool) pre = (pool - pre_first + pre_stride - 1) / pre_stride;
    }
    // Item i of a worker, or -1 after its last one.
    __device__ __forceinline__ int nth(int i, int worker, int workers) const {
        if (i < pre) return pre_first + i * pre_stride;
        const int64_t t = int64_t(pool) + worker + int64_t(i - pre) * workers;
        return t < items ? int(t) : -1;
    }
    // Item t: its tile and its share [k0, k1) of the K stages.
    __device__ __forceinline__ void item(int t, int& mb, int& nb, int& part, int& k0, int& k1) const {
        part = 0;
        k0 = 0;
        k1 = k_steps;
        if (t >= walk.whole && walk.parts > 1) {
            const int tile = walk.whole + (t - walk.whole) / walk.parts;
            part = (t - walk.whole) % walk.parts;
            k0 = min(part * part_steps, k_steps);
            k1 = min(k0 + part_steps, k_steps);
            t = tile;
        }
        walk.coords(t, mb, nb);
    }
};

// One lane of a converged warp, always the same.
__device__ __forceinline__ bool elected() {
    uint32_t is;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(is));
    return is != 0;
}

// D[tmem] (+)= A[smem] B[smem], 16-bit operands, fp32 accumulation.
template <bool kPair>
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
    if (kPair)
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
}

// Arrive on the barrier (of both CTAs of a pair) once every MMA issued so far is done.
template <bool kPair>
__device__ __forceinline__ void commit(uint32_t bar) {
    if (kPair)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                bar),
            "h"((uint16_t)3)
            : "memory");
    else
        ptx::tc_commit(bar);
}

template <bool kPair>
__device__ __forceinline__ void tmem_alloc(uint32_t slot_smem, uint32_t ncols) {
    if (kPair) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot_smem), "r"(ncols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        ptx::tmem_alloc(slot_smem, ncols);
        ptx::tmem_relinquish();
    }
}
template <bool kPair>
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    if (kPair)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols));
    else
        ptx::tmem_dealloc(taddr, ncols);
}

// A TMA load into this CTA's shared memory that completes on `bar`, which with
// kPair lies in the pair's first CTA (a shared::cluster address).
template <bool kPair>
__device__ __forceinline__ void tma_load(uint32_t dst, const void* tmap, int32_t x, int32_t y, uint32_t bar) {
    if (kPair)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
            "%3}], [%4];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        ptx::tma_load_2d(dst, tmap, x, y, bar);
}

// Adds a box of shared memory to Float32 values in global memory.
__device__ __forceinline__ void tma_add_2d(const void* tmap, int32_t x, int32_t y, uint32_t src) {
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(tmap)),
                 "r"(x), "r"(y), "r"(src)
                 : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Shared-memory address of the same variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
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

// Loads 32 consecutive Float32 TMEM columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_ld_f32_x32(uint32_t taddr, float (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr));
}

// The target entries of one row inside a half tile, a row per lane.  fetch()
// copies them into the warp's staging box while the MMAs run (the lists are
// ascending, in L2; walking them there would wait for L2 at every entry);
// walk() then runs `take` for every entry inside 32 columns held in registers.
struct EntryCursor {
    static constexpr int kHeld = 16;  // entries of a row that the box holds; more are read from the list
    const int* idx;
    const float* p;
    uint2* box;     // [kHeld][32 lanes]
    int first, n;   // the row's entries first .. first + n - 1 lie in the half tile
    int i;          // the next one
    int next;       // its column, INT_MAX past the end
    float prob;     // and probability

    __device__ __forceinline__ void fetch(const GemmArgs& a, uint8_t* warp_box, int lane, int64_t row, bool row_in,
                                          int col0, int cols) {
        idx = a.ent_idx + row * a.ent_k;
        p = a.ent_p ? a.ent_p + row * a.ent_k : nullptr;
        box = reinterpret_cast<uint2*>(warp_box) + lane;
        first = n = 0;
        if (!row_in || cols <= 0) return;
        int e = 0, end = 1;
        if (a.offs) {
            e = a.offs[int64_t(col0 / kEntryTile) * a.rows_pad + row];
            end = a.offs[int64_t((col0 + cols - 1) / kEntryTile + 1) * a.rows_pad + row];
        }
        for (; e < end; e += 4) {
            int c[4];
            float q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in = e + j < end;
                c[j] = in ? idx[e + j] : INT_MAX;
                q[j] = in && p ? p[e + j] : 1.0f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c[j] >= col0 && c[j] < col0 + cols) {
                    if (n == 0) first = e + j;
                    if (n < kHeld) box[n * 32] = make_uint2(uint32_t(c[j]), __float_as_uint(q[j]));
                    ++n;
                }
        }
    }
    __device__ __forceinline__ void load() {
        next = INT_MAX;
        prob = 0.0f;
        if (i < n) {
            if (i < kHeld) {
                const uint2 v = box[i * 32];
                next = int(v.x);
                prob = __uint_as_float(v.y);
            } else {
                next = idx[first + i];
                prob = p ? p[first + i] : 1.0f;
            }
        }
    }
    __device__ __forceinline__ void begin() {
        i = 0;
        load();
    }
    template <class F>
    __device__ __forceinline__ void walk(int chunk0, F&& take) {
        while (__any_sync(0xffffffffu, next < chunk0 + 32)) {
            const bool mine = next < chunk0 + 32;
            take(mine ? next - chunk0 : -1, prob);
            if (mine) {
                ++i;
                load();
            }
        }
    }
};

// Two values' hi parts in the type of a Float32 operand's planes; x and y keep
// what that leaves.
template <bool kWide>
__device__ __forceinline__ uint32_t split2(float& x, float& y) {
    if (kWide) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        x -= __low2float(h);
        y -= __high2float(h);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(x, y);
    x -= __low2float(h);
    y -= __high2float(h);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t split2(bool wide, float& x, float& y) {
    return wide ? split2<true>(x, y) : split2<false>(x, y);
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (kBf16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&v);
    }
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}

// What an epilogue warp knows about its 32 rows of a tile.
template <int kBoxes>
struct WarpRows {
    uint8_t* box;   // its staging boxes of 4 KiB
    int lane;
    int64_t m0;     // first row; lane holds row m0 + lane
    bool row_in;

    // Stores of 32 rows x 128 bytes through the output map: begin() waits until
    // the staging boxes are free, stage() writes a box, a row per lane in
    // registers (16-byte units swizzled by row % 8, as the map says), and
    // send() hands the boxes to TMA, at elements x0 (and x1) of row y: stored,
    // or added.  What lies outside the map is clipped.  (The proxy fence costs
    // about 1000 cycles: one for all boxes.)
    __device__ __forceinline__ void begin() {
        if (lane == 0) ptx::bulk_wait_group_read0();
        __syncwarp();
    }
    __device__ __forceinline__ void stage(int slot, const uint32_t (&w)[32]) {
        uint8_t* b = box + slot * 4096 + lane * 128;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            *reinterpret_cast<uint4*>(b + (u ^ (lane & 7)) * 16) =
                make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
    }
    __device__ __forceinline__ void send(const void* tmap, int boxes, int x0, int x1, int y, bool add) {
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            const uint32_t b = ptx::smem_addr(box);
            if (add) {
                tma_add_2d(tmap, x0, y, b);
                if (boxes > 1) tma_add_2d(tmap, x1, y, b + 4096);
            } else {
                ptx::tma_store_2d(tmap, x0, y, b);
                if (boxes > 1) ptx::tma_store_2d(tmap, x1, y, b + 4096);
            }
            ptx::bulk_commit_group();
        }
    }
    // The same for two boxes, word(b, j) of box b, at elements x0 and x1;
    // `second`: whether the second one exists.
    template <class F>
    __device__ __forceinline__ void send_two(const void* tmap, F&& word, bool second, int x0, int x1, int y, bool add) {
        uint32_t w[32];
        begin();
#pragma unroll
        for (int j = 0; j < 32; ++j) w[j] = word(0, j);
        stage(0, w);
        if (kBoxes == 1) send(tmap, 1, x0, 0, y, add);
        if (second) {
            if (kBoxes == 1) begin();
#pragma unroll
            for (int j = 0; j < 32; ++j) w[j] = word(1, j);
            stage(kBoxes - 1, w);
        }
        if (kBoxes > 1) send(tmap, second ? 2 : 1, x0, x1, y, add);
        else if (second) send(tmap, 1, x1, 0, y, add);
    }
};

// Softmax statistics of a row over the half tile in registers, of z = h w =
// r inv: top = max z, sum of exp2(k2 (z - top)), target term sum p z.  What follows
// starts from differences of z: a rounded k2 z of 60 is off by 2^-18, of which a
// row sure of its target has nothing left.  The exponentials'
// fma takes the rounded k2 top off, and what that rounding left is a factor of the
// row (1400 x 50001, dim 2048: 206.6 us; subtracting z first 210); only where it
// would be large (logits above 10^6) the difference comes first.  With `keep` the
// exponentials are stored too, for the gradient: as f16 times 2^15 (11 bits down
// to 2^-29 of the half tile's largest; the later rounding to bf16 is the one
// that counts) or, for Float32, as they are.
template <bool kBf16, int kBlocks, class Rows>
__device__ __forceinline__ float4 lse_tile(const GemmArgs& args, const void* tmap_c, Rows& wr, EntryCursor& cur,
                                           int64_t n0, int64_t n_end, float inv, float (&r)[kBlocks][2][32]) {
    const int64_t m = wr.m0 + wr.lane;
    float top = -INFINITY, dot = 0.0f;
#pragma unroll
    for (int c = 0; c < 2 * kBlocks; ++c) {
        cur.walk(int(args.v0 + n0) + c * 32, [&](int rel, float p) {
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j == rel) v = r[c / 2][c % 2][j];
            if (rel >= 0) {
                if (p != 0.0f) dot += p * v;
                if (args.ent_s) args.ent_s[m * args.ent_k + cur.first + cur.i] = v * inv;
            }
        });
        const int ncols = (int)min(int64_t(32), n_end - (n0 + c * 32));
        if (ncols < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j >= ncols) r[c / 2][c % 2][j] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) top = fmaxf(top, r[c / 2][c % 2][j]);
    }
    // columns of nothing but -inf add nothing (and must not make -inf minus -inf)
    const float base = top == -INFINITY ? 0.0f : top;
    const float k2 = args.logit_scale * kLog2e * inv;
    float sum = 0.0f, ref = __fmul_rn(base, k2), rest = fmaf(base, k2, -ref);
    if (__builtin_expect(!(fabsf(ref) < kLargeExponent), 0)) {
#pragma unroll
        for (int c = 0; c < 2 * kBlocks; ++c)
#pragma unroll
            for (int j = 0; j < 32; ++j) r[c / 2][c % 2][j] -= base;
        ref = rest = 0.0f;
    }
    const float fix = ex2(-rest);
#pragma unroll
    for (int c = 0; c < 2 * kBlocks; ++c) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            r[c / 2][c % 2][j] = ex2(fmaf(r[c / 2][c % 2][j], k2, -ref));
            sum += r[c / 2][c % 2][j];
        }
    }
    if (args.keep && n0 < n_end) {  // (blocks of 64 columns are written whole)
        const float up = !wr.row_in ? 0.0f : kBf16 ? 32768.0f * fix : fix;
        if (kBf16) {
            wr.send_two(
                tmap_c,
                [&](int b, int j) {
                    const float (&x)[32] = r[b][j / 16];
                    return pack2<false>(x[2 * (j % 16)] * up, x[2 * (j % 16) + 1] * up);
                },
                n0 + 64 < n_end, int(n0), int(n0) + 64, int(wr.m0), false);
        } else {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
                if (n0 + b * 64 < n_end)
                    wr.send_two(
                        tmap_c, [&](int c, int j) { return __float_as_uint(r[b][c][j] * up); }, true,
                        2 * (int(n0) + b * 64), 2 * (int(n0) + b * 64 + 32), int(wr.m0), false);
        }
    }
    return make_float4(top * inv, sum * fix, dot * inv, 0.0f);
}

// What a row's logits' gradient needs: (exp2(k2 z - ref) - p fix) coef.
struct SoftmaxRow {
    float ref, fix, coef;

    __device__ __forceinline__ SoftmaxRow() : ref(0.0f), fix(1.0f), coef(0.0f) {}
    __device__ __forceinline__ void load(const GemmArgs& args, int64_t m, float gscale) {
        const float2 norm = args.norm[m];
        const float top = __fmul_rn(norm.x, args.to_log2);
        ref = top + norm.y;
        const float part = ref - top;  // (the sum and its rounding error, exactly)
        const float rest = fmaf(norm.x, args.to_log2, -top) + ((top - (ref - part)) + (norm.y - part)) -
                           norm.x * args.factor_rest;
        const bool large = !(fabsf(ref) < kLargeExponent);
        fix = large ? 1.0f : ex2(rest);
        coef = args.coef[m] * gscale * (large ? 1.0f : ex2(-rest));
    }
};

// Gradient with respect to the logits of a half tile's row: softmax minus
// target in fp32, rounded once to the type the next contractions read.  As
// above, what rounding the exponent's constant left is a factor of the row.
template <bool kBf16, bool kFew, class Rows>
__device__ __forceinline__ void grad_tile(const GemmArgs& args, const void* tmap_c, Rows& wr, EntryCursor& cur,
                                          int64_t n0, int64_t n_end, float inv, const SoftmaxRow& row, bool wide,
                                          float (&r)[2][2][32]) {
    if (n0 >= n_end || (kFew && wr.m0 >= kFewRows)) return;  // (the remainders' rows are written below)
    float k2 = args.logit_scale * kLog2e * inv, ref = row.ref;
    if (__builtin_expect(!(fabsf(ref) < kLargeExponent), 0)) {
        const float2 norm = args.norm[wr.m0 + wr.lane];  // (a row that exists: others have ref 0)
        const float to_ref = args.to_ref * inv;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 32; ++j)
                r[c / 2][c % 2][j] = __fsub_rn(__fmul_rn(r[c / 2][c % 2][j], to_ref), norm.x);
        k2 = args.to_log2;
        ref = norm.y;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        float (&x)[32] = r[c / 2][c % 2];
        const int ncols = (int)min(int64_t(32), n_end - (n0 + c * 32));
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = ex2(fmaf(x[j], k2, -ref));
        cur.walk(int(args.v0 + n0) + c * 32, [&](int rel, float p) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j == rel) x[j] -= p * row.fix;
        });
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] *= row.coef;  // (0 in a row that does not exist)
        if (ncols < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j >= ncols) x[j] = 0.0f;
        }
    }
    if (kBf16) {
        wr.send_two(
            tmap_c,
            [&](int b, int j) {
                float& x = r[b][j / 16][2 * (j % 16)];
                float& y = r[b][j / 16][2 * (j % 16) + 1];
                const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
                if (kFew) {  // what the rounding leaves
                    x -= __low2float(h);
                    y -= __high2float(h);
                }
                return *reinterpret_cast<const uint32_t*>(&h);
            },
            n0 + 64 < n_end, int(n0), int(n0) + 64, int(wr.m0), false);
        if (kFew)
            wr.send_two(
                tmap_c,
                [&](int b, int j) { return pack2<true>(r[b][j / 16][2 * (j % 16)], r[b][j / 16][2 * (j % 16) + 1]); },
                n0 + 64 < n_end, int(n0), int(n0) + 64, int(wr.m0) + kFewRows, false);
    } else {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if (n0 + b * 64 >= n_end) continue;
            // (the second plane from what the first one leaves)
            const int x0 = 2 * (int(n0) + b * 64);
            if (wide)
                wr.send_two(
                    tmap_c,
                    [&](int, int j) { return split2<true>(r[b][j / 16][2 * (j % 16)], r[b][j / 16][2 * (j % 16) + 1]); },
                    true, x0, x0 + 64, int(wr.m0), false);
            else
                wr.send_two(
                    tmap_c,
                    [&](int, int j) { return split2<false>(r[b][j / 16][2 * (j % 16)], r[b][j / 16][2 * (j % 16) + 1]); },
                    true, x0, x0 + 64, int(wr.m0), false);
        }
    }
}

// A half tile of a result, through the output map: into fp32 running sums (row
// y of the map is this part's row) or in the result's type.
template <bool kF32, class Rows>
__device__ __forceinline__ void out_tile(const Problem& args, const void* tmap_c, Rows& wr, int y, int64_t n0,
                                         float scale, float (&r)[2][2][32]) {
    if (n0 >= args.N) return;
    if (kF32 || args.sums) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int x = int(n0) + b * 64;
            if (x < args.N)
                wr.send_two(
                    tmap_c,
                    [&](int c, int j) { return __float_as_uint(r[b][c][j] * scale); },
                    x + 32 < args.N, x, x + 32, y, args.sums && !args.first);
        }
    } else {
        wr.send_two(
            tmap_c,
            [&](int b, int j) {
                return pack2<true>(r[b][j / 16][2 * (j % 16)] * scale, r[b][j / 16][2 * (j % 16) + 1] * scale);
            },
            n0 + 64 < args.N, int(n0), int(n0) + 64, y, false);
    }
}

// The contraction kernel.  A launch computes args.p[0] (kBoth: and args.p[1], half
// of the workers each first, see Plan).  The tensor cores bound it, and under
// long load the power limit; a tile's epilogue runs under the next tile's MMAs:
//
//   4096 x 32000, dim 4096: logits with statistics and their exponentials 710 us
//   (tensor pipe 91 % busy), dh 694 (93 %), dw 686 (91 %): 1.51, 1.55, 1.57 PFLOP/s;
//   3891 rows, dim 2048: 430 (76 %), 349 (96 %), 326 (89 %).  The logits of short walks
//   stay behind: at dim 1024 a 256 x 256 tile lasts about 10000 cycles, its epilogue
//   5400, with the exponentials' store 9500.
//   Float32, 2048 x 32000, dim 1024, three plane pairs: 308 (75 %), 295 (88 %), 301
//   (75 %): 1.31, 1.36, 1.34 PFLOP/s of f16 products.
//   1 x 32000, dim 4096: 52 us, the read of w at 5.0 TB/s; 64 x 131072, dim 2048:
//   105 us, 5.1 TB/s, both gradients in one launch 208 us, 5.2 TB/s.
template <int kShape, bool kBf16, int kEpi, int kA>
__global__ void __launch_bounds__(320, 1)
    head_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ GemmArgs args) {
    constexpr bool kBMn = kEpi == kEpiOut;  // logits contract K-major operands
    constexpr bool kGrad = kEpi == kEpiGrad || kEpi == kEpiGradCut;
    constexpr int kProblems = kA == kBoth ? 2 : 1;
    auto mn_major = [](const Problem& p) { return kA == kBoth ? p.a_mn != 0 : kA == kMnMajor; };
    using C = Cfg<kShape>;
    constexpr bool kPair = C::kPair;
    constexpr bool kChunked = !kBf16 || kEpi == kEpiLse || kEpi == kEpiGradCut;
    static_assert(C::kAccs == 1 || !kChunked, "the tall tile has no accumulator to alternate with");
    constexpr int kStages = C::kStages;
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
    // of a pair, the first CTA holds the barriers that the MMA thread waits on
    const uint32_t rank = kPair ? cluster_rank() : 0;
    const int worker = kPair ? blockIdx.x >> 1 : blockIdx.x, workers = kPair ? gridDim.x >> 1 : gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(bar_full + 8 * s, 1);
            ptx::mbar_init(bar_empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            ptx::mbar_init(bar_tmem_full + 8 * b, 1);
            ptx::mbar_init(bar_tmem_empty + 8 * b, kPair ? 16 : 8);  // a lane of every epilogue warp
        }
        ptx::mbar_init(bar_drain, 1);
        ptx::fence_barrier_init();
        for (int q = 0; q < args.problems; ++q) {
            ptx::prefetch_tmap(&maps.a[q]);
            ptx::prefetch_tmap(&maps.b[q]);
            if (kGrad || kEpi == kEpiOut || args.keep) ptx::prefetch_tmap(&maps.c[q]);
        }
    }
    if (warp == 1) tmem_alloc<kPair>(ptx::smem_addr(tmem_slot), C::kTmemCols);
    ptx::tc_fence_before();
    __syncthreads();
    __syncwarp();
    if (kPair) cluster_sync();  // the other CTA's barriers are initialised
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_enter();

    constexpr bool kNarrow = kShape == kSingle && kEpi != kEpiOut;  // tiles may be narrower
    const int tile_n = kNarrow ? args.tile_n : kBN;
    // rows that count, and for the gradients of few rows their remainders
    const bool few = kBf16 && kEpi != kEpiLse && args.state->few(args.row0);
    const bool wide = !kBf16 && args.state->wide;
    const Products pairs = products(!kBf16, wide, kEpi == kEpiOut);
    auto plan_of = [&](const Problem& p) {
        int rows = args.state->rows(args.row0);
        if (!few) rows = min(rows, p.count_is == kCountM ? p.M : p.K);
        else if (kEpi == kEpiOut) rows += kFewRows;
        return Plan(p.count_is == kCountM ? rows : p.M, p.N, p.count_is == kCountK ? rows : p.K, C::kTileM, tile_n,
                    workers,
                    p.splits > 0 ? p.splits : args.state->dh_splits);
    };
    const Plan plan0 = plan_of(args.p[0]);
    Plan plan1 = plan0;
    if (kProblems > 1 && args.problems > 1) {
        plan1 = plan_of(args.p[1]);
        plan1.follow(plan0, worker, workers, stage_us(kShape, args.terms), fixed_us(kShape));
    }
    // Reading the weights for the one and writing the other is what a call of
    // few rows does: half of the workers at a time do each.
    const int flip = kProblems > 1 && args.problems > 1 && args.alternate && (worker & 1);
    // Columns that the MMAs of column tile `nb` compute: whole 64s of what is left
    // of a result (a dim of 64 or 320 would waste three quarters of a tile).
    auto tile_cols = [&](const Problem& p, int nb) {
        return kEpi == kEpiOut ? min(kBN, (p.N - nb * kBN + 63) / 64 * 64) : tile_n;
    };
    auto chunk_end = [&](int k0, int k1) { return kChunked ? min(k0 + args.chunk, k1) : k1; };

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- producer ----------------
            int stage = 0;
            uint32_t phase = 0;
            uint32_t issued[kStages] = {0};
            bool alive = true;
            for (int ph = 0; ph < (kProblems > 1 ? args.problems : 1) && alive; ++ph) {
                const int q = kProblems > 1 ? ph ^ flip : 0;
                const Plan plan = kProblems > 1 && q ? plan1 : plan0;
                const Problem& p = args.p[q];
                const CUtensorMap *ma = &maps.a[q], *mb_ = &maps.b[q];
                const bool a_mn = mn_major(p);
                for (int i = 0, t; alive && (t = plan.nth(i, worker, workers)) >= 0; ++i) {
                    int mb, nb, split, k0, k1;
                    plan.item(t, mb, nb, split, k0, k1);
                    const int b_cols = tile_cols(p, nb) / (kPair ? 2 : 1);  // of this CTA
                    const int boxes = (b_cols + 63) / 64;
                    const int a0 = mb * C::kTileM + rank * kBM, b0 = nb * tile_n + rank * b_cols;
                    const uint32_t bytes =
                        (kPair ? 2 : 1) * (C::kABytes + (kEpi == kEpiOut ? boxes * 64 : b_cols) * kBK * 2);
                    for (int c0 = k0; c0 < k1 && alive; c0 = chunk_end(c0, k1))
                        for (int term = 0; term < pairs.terms && alive; ++term) {
                            const int pa = plane_of(pairs.a, term), pb = plane_of(pairs.b, term);
                            const int xa = pa * p.pa.x_plane, ya = pa * p.pa.y_plane;
                            const int xb = pb * p.pb.x_plane, yb = pb * p.pb.y_plane;
                            const int c1 = chunk_end(c0, k1);
                            for (int ks = c0; ks < c1; ++ks) {
                                if (!ptx::mbar_wait(bar_empty + 8 * stage, phase ^ 1)) { alive = false; break; }
                                const uint32_t own = bar_full + 8 * stage;
                                const uint32_t full = kPair ? mapa(own, 0) : own;
                                const uint32_t sa = sbase + stage * C::kStageBytes;
                                const uint32_t sb = sa + C::kABytes;
                                // the first CTA's barrier counts both CTAs' bytes
                                if (rank == 0) ptx::mbar_arrive_expect_tx(own, bytes);
#pragma unroll
                                for (int h = 0; h < C::kAccs; ++h) {
                                    const uint32_t sah = sa + h * (kBM * kBK * 2);
                                    const int ah = a0 + h * C::kAccRows;
                                    // (an MN-major map's boxes are 64 x 64, a K-major one's 64 x 128)
                                    if (a_mn) {
#pragma unroll
                                        for (int g = 0; g < kBM / 64; ++g)
                                            tma_load<kPair>(sah + g * 8192, ma, (ah / 64 + g) * p.pa.x_block + xa,
                                                            ya + ks * kBK, full);
                                    } else {
                                        tma_load<kPair>(sah, ma, ks * p.pa.x_block + xa, ya + ah, full);
                                    }
                                }
                                if (kBMn) {
                                    // (B's planes lie below each other: its columns are as in memory)
                                    for (int g = 0; g < boxes; ++g)
                                        tma_load<kPair>(sb + g * 8192, mb_, b0 + g * 64, yb + ks * kBK, full);
                                } else {
                                    tma_load<kPair>(sb, mb_, ks * p.pb.x_block + xb, yb + b0, full);
                                }
                                issued[stage] += 1;
                                if (++stage == kStages) { stage = 0; phase ^= 1; }
                            }
                        }
                }
            }
            // Let every copy land, and every MMA's release of a stage arrive,
            // before this CTA (and the pair) can exit.
            for (int s = 0; s < kStages; ++s)
                if (issued[s] > 0) {
                    if (rank == 0) ptx::mbar_wait(bar_full + 8 * s, (issued[s] - 1) & 1);
                    if (alive) ptx::mbar_wait(bar_empty + 8 * s, (issued[s] - 1) & 1);
                }
        }
    } else if (warp == 1) {
        // (the whole warp keeps in step and one lane issues)
        if (rank == 0) {
            // ---------------- MMA issuer ----------------
            int stage = 0;
            uint32_t phase = 0, it = 0;
            bool alive = true;
            for (int ph = 0; ph < (kProblems > 1 ? args.problems : 1) && alive; ++ph) {
                const int q = kProblems > 1 ? ph ^ flip : 0;
                const Plan plan = kProblems > 1 && q ? plan1 : plan0;
                const bool a_mn = mn_major(args.p[q]);
                // K-major: 16 elements of K are 32 bytes of the swizzled row, 8-row groups 1024 bytes apart.
                // MN-major: 16 rows of K are 2048 bytes, 64-element blocks of the other mode 8192 bytes
                // apart, 8-row groups of K 1024.  Descriptors count in 16 bytes, and the stages
                // stay below 2^18: each is the first one plus an offset.
                const uint32_t a_step = a_mn ? 2048 / 16 : 32 / 16, b_step = kBMn ? 2048 / 16 : 32 / 16;
                const uint64_t a_desc = ptx::smem_desc(sbase, a_mn ? 8192 : 0, 1024, ptx::kLayoutSwizzle128);
                const uint64_t b_desc =
                    ptx::smem_desc(sbase + C::kABytes, kBMn ? 8192 : 0, 1024, ptx::kLayoutSwizzle128);
                for (int i = 0, t; alive && (t = plan.nth(i, worker, workers)) >= 0; ++i) {
                    int mb, nb, split, k0, k1;
                    plan.item(t, mb, nb, split, k0, k1);
                    const uint32_t idesc = idesc_f16(kBf16 || wide, a_mn, kBMn, C::kAccRows, tile_cols(args.p[q], nb));
                    for (int c0 = k0; c0 < k1 && alive; c0 = chunk_end(c0, k1), ++it) {
                        // one tile alternates between the two accumulators, a tall one fills both
                        const uint32_t buf0 = C::kAccs == 1 ? it & 1 : 0;
                        const uint32_t drained = (C::kAccs == 1 ? it >> 1 : it) & 1;
                        const int steps = (chunk_end(c0, k1) - c0) * pairs.terms;
                        for (int ks = 0; ks < steps && alive; ++ks) {
                            alive = __all_sync(0xffffffffu, ptx::mbar_wait(bar_full + 8 * stage, phase));
                            if (!alive) break;
                            ptx::tc_fence_after();
#pragma unroll
                            for (int h = 0; h < C::kAccs; ++h) {
                                const uint32_t buf = buf0 + h;
                                if (ks == 0) {
                                    alive = __all_sync(0xffffffffu,
                                                       ptx::mbar_wait(bar_tmem_empty + 8 * buf, drained ^ 1));
                                    if (!alive) break;
                                    ptx::tc_fence_after();
                                }
                                const uint32_t acc = tmem + buf * kBN;
                                const uint64_t ad =
                                    a_desc + uint32_t(stage * C::kStageBytes + h * (kBM * kBK * 2)) / 16;
                                const uint64_t bd = b_desc + uint32_t(stage * C::kStageBytes) / 16;
                                if (elected()) {
#pragma unroll
                                    for (int j = 0; j < kBK / 16; ++j)
                                        mma_f16<kPair>(acc, ad + a_step * j, bd + b_step * j, idesc,
                                                       (ks > 0 || j > 0) ? 1u : 0u);
                                    if (C::kAccs > 1 && ks + 1 == steps) commit<kPair>(bar_tmem_full + 8 * buf);
                                }
                            }
                            if (!alive) break;
                            if (elected()) commit<kPair>(bar_empty + 8 * stage);
                            if (++stage == kStages) { stage = 0; phase ^= 1; }
                        }
                        if (!alive) break;
                        if (C::kAccs == 1 && elected()) commit<kPair>(bar_tmem_full + 8 * buf0);
                    }
                }
            }
            // every MMA is done before TMEM is released
            if (elected()) commit<kPair>(bar_drain);
            ptx::mbar_wait(bar_drain, 0);
        }
    } else {
        // ---------------- epilogue ----------------
        constexpr int kCols = kBN / 2;  // columns of this warp: half of the tile
        const int quarter = warp & 3;
        const int half = (warp - 2) >> 2;
        WarpRows<C::kBoxes> wr;
        wr.box = smem + C::kOffOut + (warp - 2) * C::kBoxes * 4096;
        wr.lane = lane;
        // inverse of the operands' power-of-two scales
        auto inverse = [&](const Problem& p) {
            float inv = 1.0f;
            if (p.scale_a >= 0) inv *= pow2i(-scale_exponent(args.state->amax[p.scale_a], wide));
            if (p.scale_b >= 0) inv *= pow2i(-scale_exponent(args.state->amax[p.scale_b], wide));
            return inv;
        };
        const float inv = inverse(args.p[0]);
        const float gscale = kGrad && !kBf16 ? pow2i(scale_exponent(args.state->amax[2], wide)) : 1.0f;
        auto release = [&](uint32_t buf) {
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (kPair) arrive_cluster(mapa(bar_tmem_empty + 8 * buf, 0));
                else ptx::mbar_arrive(bar_tmem_empty + 8 * buf);
            }
        };
        uint32_t it = 0;
        bool alive = true;
        for (int ph = 0; ph < (kProblems > 1 ? args.problems : 1) && alive; ++ph) {
            const int q = kProblems > 1 ? ph ^ flip : 0;
            const Plan plan = kProblems > 1 && q ? plan1 : plan0;
            const Problem& p = args.p[q];
            const void* tmap_c = &maps.c[q];
            const int M = kEpi == kEpiOut ? 0 : min(args.state->rows(args.row0), few ? INT_MAX : p.M);
            const float out_scale = kEpi == kEpiOut ? inverse(p) * args.state->grad_scale : 1.0f;
            for (int i = 0, t; alive && (t = plan.nth(i, worker, workers)) >= 0; ++i) {
                int mb, nb, split, k0, k1;
                plan.item(t, mb, nb, split, k0, k1);
#pragma unroll 1
                for (int h = 0; h < C::kAccs && alive; ++h) {
                    wr.m0 = int64_t(mb) * C::kTileM + h * C::kAccRows + rank * kBM + quarter * 32;
                    const int64_t m = wr.m0 + lane;
                    wr.row_in = m < M;
                    const int64_t ncol0 = int64_t(nb) * tile_n + half * kCols;
                    const int64_t n_end = min(int64_t(p.N), min(ncol0 + kCols, int64_t(nb + 1) * tile_n));
                    // a pair's second half may lie past the rows that the workspace holds
                    // (and a narrow tile's second half is none)
                    const bool rows_in = kEpi == kEpiOut || (wr.m0 < (p.M + kBM - 1) / kBM * kBM &&
                                                             (!kNarrow || half * kCols < tile_n));
                    // what the row needs beside its accumulator, while the MMAs run
                    EntryCursor cur;
                    SoftmaxRow row;
                    if (kEpi != kEpiOut) {
                        wr.begin();  // the entries go where the stores' boxes are
                        cur.fetch(args, wr.box, lane, m, wr.row_in, int(args.v0 + ncol0), int(n_end - ncol0));
                    }
                    if (kGrad && wr.row_in) row.load(args, m, gscale);
                    const uint32_t lanes = uint32_t(quarter * 32) << 16;
                    // The half tile's row in registers: the accumulator is free again
                    // before any of the work on it.  (An empty share of K: zeros.)
                    float r[2][2][32];
                    if (k0 >= k1) {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int j = 0; j < 32; ++j) r[c / 2][c % 2][j] = 0.0f;
                    }
                    for (int c0 = k0; c0 < k1; c0 = chunk_end(c0, k1)) {
                        const uint32_t buf = C::kAccs == 1 ? it & 1 : h, filled = (C::kAccs == 1 ? it >> 1 : it) & 1;
                        if (!__all_sync(0xffffffffu, ptx::mbar_wait(bar_tmem_full + 8 * buf, filled))) {
                            alive = false;
                            break;
                        }
                        ptx::tc_fence_after();
                        const uint32_t acc = tmem + buf * kBN + half * kCols + lanes;
                        if (c0 == k0) {
#pragma unroll
                            for (int c = 0; c < 4; ++c) tmem_ld_f32_x32(acc + c * 32, r[c / 2][c % 2]);
                            ptx::tmem_ld_wait();
                        } else if (kChunked) {
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                uint32_t u[16];
                                tmem_ld_32x32b_x16(acc + c * 16, u);
                                ptx::tmem_ld_wait();
#pragma unroll
                                for (int j = 0; j < 16; ++j)
                                    r[c / 4][c / 2 % 2][c % 2 * 16 + j] += __uint_as_float(u[j]);
                            }
                        }
                        release(buf);
                        if (h + 1 == C::kAccs) ++it;
                    }
                    if (!alive) break;
                    if (!rows_in) continue;
                    if (kEpi != kEpiOut) cur.begin();
                    if (kEpi == kEpiLse) {
                        const float4 st = lse_tile<kBf16, 2>(args, tmap_c, wr, cur, ncol0, n_end, inv, r);
                        args.partial[m * args.slots + ((args.v0 + ncol0) >> args.slot_shift)] = st;
                    } else if (kGrad) {
                        if (few) grad_tile<kBf16, kBf16>(args, tmap_c, wr, cur, ncol0, n_end, inv, row, wide, r);
                        else grad_tile<kBf16, false>(args, tmap_c, wr, cur, ncol0, n_end, inv, row, wide, r);
                    } else {
                        const int y = p.sums ? plan.walk.sum_row(split, int(wr.m0)) : int(wr.m0);
                        out_tile<!kBf16>(p, tmap_c, wr, y, ncol0, out_scale, r);
                    }
                }
            }
        }
        if (lane == 0) ptx::bulk_wait_group0();  // this warp's stores are done
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (kPair) {
        // the MMA thread's last commit arrives in the second CTA too: not after it has left
        if (rank == 1 && threadIdx.x == 0) ptx::mbar_wait(bar_drain, 0);
        __syncwarp();
        cluster_sync();
    }
    ptx::tc_fence_after();
    if (warp == 1) tmem_dealloc<kPair>(tmem, C::kTmemCols);
}

}  // namespace head
}  // namespace sw
