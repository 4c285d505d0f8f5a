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
// the contractions of sw_head_gemm.cuh then run over the compact rows.
//
// A loss: the logits' tiles leave a (max, sum, target term) triple per row and
// half tile, and loss_kernel adds them up: 2 T V D operations, no logits held.
//
// A loss with gradients in one call: the tiles also leave exp2(s - max) of
// their own maxima, 16 bits each (Float32: 32), loss_kernel turns them into G
// in place once it knows the row's sum, and two contractions take G to dh and
// dw: 6 T V D and one pass over T V values.  That pass costs 110 us of the
// 1464 of 4096 x 32000 x 2048; computing the logits again 430.  Where the
// workspace limit holds fewer rows, the rows go in blocks, dh and dw added up
// in fp32.
//
// Gradients from a kept lse (or below that limit): the logits of a piece of the
// vocabulary are computed (again), their gradient is rounded once to the operand
// type in the epilogue, and the two contractions follow, piece by piece: 8 T V D
// with the loss, 6 without.
//
// bf16 operands are used as they are.  A common factor of all rows (a mean's, an
// upstream gradient's) is left out of the 16-bit G and put to the results in
// fp32, so that a target's -1 is exact; with at most 64 rows that count, what
// the rounding of G left goes along as further rows, for nothing averages it
// out there.
//
// What bounds it: the contractions on the tensor cores, under the power limit
// for the large steps (8192 x 131072 x 4096: 21.1 ms on a GPU that runs a
// library's three products alone in 19.1, and 2.71 against 2.39 ms at 4096 x
// 32000 x 4096); for few rows the bytes of w (64 x 131072 x 2048: 405 us for two
// reads and a write of it, 4.0 TB/s).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <numeric>
#include <type_traits>

#include "sw_common.cuh"
#include "sw_head_rows.cuh"
#include "sw_ptx.cuh"
#include "sw_tma.cuh"

namespace sw {
namespace head {
namespace {

// What a call may take unless the plan says otherwise: the exponentials of 16384
// rows over a vocabulary of 131072 are half of it.
constexpr int64_t kDefaultWorkspace = int64_t(8) << 30;

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

// How a contraction is spread over the SMs: the parts of the K walk that suit a
// tile shape, and the estimate.  `sum_us`: what it costs more to go through fp32
// sums when nothing else asks for them.
struct Spread {
    int splits;
    float us;
};
Spread choose_parts(int64_t M, int64_t N, int64_t K, int terms, int shape, bool may_split, float sum_us = 0.0f) {
    Spread best{1, 1e30f};
    for (int s = 1; s <= (may_split ? kMaxParts : 1); ++s) {
        const float us = spread_cost(M, N, K, terms, shape, device_sms(), s) + (s > 1 ? sum_us : 0.0f);
        if (us < best.us * 0.97f) best = Spread{s, us};
    }
    return best;
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

// The operands and the result of one contraction.
struct Tensors {
    Operand a, b;
    Target c;
};

template <int kShape, bool kBf16, int kEpi, int kA>
int launch_gemm(const Tensors* t, GemmArgs& args, cudaStream_t stream) {
    using Cf = Cfg<kShape>;
    Maps maps;
    memset(&maps, 0, sizeof(maps));
    for (int q = 0; q < args.problems; ++q) {
        // boxes of K-major operands are 64 wide and as high as a CTA's share of
        // the tile, of MN-major ones 64 x 64
        Problem& p = args.p[q];
        int rc = make_map(&maps.a[q], t[q].a.ptr, t[q].a.rows, t[q].a.cols, t[q].a.ld, p.a_mn ? kBK : kBM);
        if (rc == SW_OK)
            rc = make_map(&maps.b[q], t[q].b.ptr, t[q].b.rows, t[q].b.cols, t[q].b.ld,
                          kEpi == kEpiOut ? kBK : kShape == kSingle ? args.tile_n : Cf::kBRows);
        if (rc == SW_OK && t[q].c.ptr) rc = make_target_map(&maps.c[q], t[q].c);
        if (rc != SW_OK) return rc;
        p.pa = t[q].a.plane;
        p.pb = t[q].b.plane;
    }
    auto kernel = head_gemm_kernel<kShape, kBf16, kEpi, kA>;
    static bool configured[64] = {};  // per device: the attribute stays
    int dev = 0;
    SW_CUDA_TRY(cudaGetDevice(&dev), "cudaGetDevice");
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        SW_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cf::kSmemBytes),
                    "linear head smem");
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    constexpr int kCtas = Cf::kPair ? 2 : 1;
    // every SM, unless it is known here that there are fewer tiles
    int64_t items = device_sms() / kCtas;
    if (args.problems == 1 && args.p[0].splits == 1)
        items = std::min<int64_t>(items, (args.p[0].M + Cf::kTileM - 1) / Cf::kTileM *
                                             ((args.p[0].N + (kEpi == kEpiOut ? kBN : args.tile_n) - 1) /
                                              (kEpi == kEpiOut ? kBN : args.tile_n)));
    if (items == 0) return SW_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kCtas * (unsigned)items);
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
    cfg.numAttrs = Cf::kPair ? 2 : 1;
    SW_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, maps, args), "linear head contraction");
    return SW_OK;
}

// K stages between two sums in registers: what the accumulator drops grows with
// them, and each costs the epilogue about 500 cycles, for which a tile's MMAs may
// have to wait.  Float32 results: 8 (at 4 a step of 2048 x 32000 at dim 1024 takes
// 1335 us, not 1300).  Logits are exponents: what they are off by is the relative
// error of a softmax.  Float32: 4 (gradients of 4663 x 1191, dim 576, off by 1.4e-6,
// at 8 by 2.9e-6; that step 1303 us against 1290), for one row tile 2 (no slower;
// 1 takes 348 us where 2 take 307, 5 x 8197 at dim 3802), and two pieces at least.
// bf16: 16 (the loss of 1400 x 50001 off by 7e-7); for one row tile, whose errors
// less averages out and which the read of w bounds, 8 (64 x 131072 with gradients 4
// us of 397 more, 4 stages 12), or 2 where no exponentials are written (one token's
// loss, over 40 inputs, off by 3.1e-6 at most, as a plain Float32 product's by 5.4e-6;
// at 16 one of them by 1.1e-5, in the same time).  The same for the logits of a
// gradient from a kept lse as for the loss that left it: both drift alike.
int chunk_stages(bool bf16, int epi, const GemmArgs& args) {
    const Problem& p = args.p[0];
    if (epi == kEpiOut) return 8;
    if (!bf16) return std::min(p.M > kBM ? 4 : 2, std::max(1, (p.K + 2 * kBK - 1) / (2 * kBK)));
    return p.M > kBM ? 16 : args.keep ? 8 : 2;
}

// One contraction, or the gradients' two in one launch (kBoth, single CTAs' tiles).
template <bool kBf16, int kEpi, int kA>
int gemm(const Tensors* t, GemmArgs& args, int shape, cudaStream_t stream) {
    args.terms = kBf16 ? 1 : 3;
    args.chunk = chunk_stages(kBf16, kEpi, args);
    if (kA == kBoth || shape == kSingle) return launch_gemm<kSingle, kBf16, kEpi, kA>(t, args, stream);
    // results summed in registers (Float32, and the statistics) have no tall tile,
    // and the logits' gradient has too much to do after a tile (4096 x 32000, dim
    // 1024 / 2048 / 4096: 242 / 395 / 719 us against 201 / 362 / 695)
    constexpr int kMost = kA == kBoth ? kSingle : kBf16 && kEpi == kEpiOut ? kTall : kPair2;
    constexpr int kMiddle = kA == kBoth ? kSingle : kPair2;
    return shape == kTall ? launch_gemm<kMost, kBf16, kEpi, kA>(t, args, stream)
                          : launch_gemm<kMiddle, kBf16, kEpi, kA>(t, args, stream);
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
    float2* norm;
    float* row_loss;
    float* ent_s;
    uint16_t* hc;
    uint32_t* row_top;
    float4* partial;
    float* dh_sums;
    float* dw_sums;
    void* dw_rows;
    uint16_t* wp;
    uint16_t* grad;
};

struct Shape {
    int64_t T, D, V, rows_pad, ld_h;
    int tile_n;              // columns of a logits tile
    int64_t slots;           // pieces of the vocabulary's tiles with statistics of their own
    int slot_shift;
    bool f32, pack_w, grads, flags;
    int planes;              // 16-bit planes of the logits' gradient: 1, Float32 2
    int op_planes;           // of the states and packed weights, at most: 1, Float32 3
    int h_parts, w_parts;    // of a row, where contiguous columns are measured by row
    // words that measuring in parts takes: a row's magnitude, a count for 32 rows
    static int64_t measured(int64_t rows, int parts) { return parts > 1 ? rows + (rows + 31) / 32 : 0; }
    int64_t row_tops() const { return measured(T, h_parts) + measured(V, w_parts); }
    // Gradients: `keep`: the forward's exponentials of `rows` compact rows at a
    // time stay in the workspace and become the logits' gradient.  Otherwise
    // the logits are computed again, `piece` columns of the vocabulary at a
    // time.  Packed weights are laid out `piece` columns at a time too.
    // A loss alone takes its statistics stat_rows compact rows at a time.
    bool keep;
    int64_t rows, piece, stat_rows;
    // Few rows (one row tile): the gradients' contractions share a launch, which
    // reads the weights while it writes their gradient.
    bool together;
    int logits_shape, dh_shape, dw_shape, dw_splits;
    // rows of fp32 sums of each gradient (0: it is written at once); dh's rows
    // are always put in place from sums, whose parts are chosen on the device
    int64_t dh_sum_rows, dw_sum_rows, ld_acc;
    // dw goes to rows padded to 16 bytes first, in its own type (TMA cannot write
    // it where it belongs)
    bool dw_padded;
};

Layout lay_out(Bump& b, const Call& c, const Shape& s) {
    Layout l;
    memset(&l, 0, sizeof(l));
    const int64_t K = c.targets ? 1 : c.top_k;
    l.state = b.take<HeadState>(1);
    l.row_map = b.take<int>(s.T);
    l.ent_idx = b.take<int>(s.rows_pad * K);
    if (!c.targets) {
        if (s.flags) l.flags = b.take<uint8_t>(s.T);
        l.ent_p = b.take<float>(s.rows_pad * K);
        l.entropy = b.take<float>(s.rows_pad);
        l.offs = b.take<uint16_t>(s.rows_pad * ((s.V + kEntryTile - 1) / kEntryTile + 1));
    }
    l.coef = b.take<float>(s.rows_pad);
    l.norm = b.take<float2>(s.rows_pad);
    l.row_loss = b.take<float>(s.rows_pad);
    l.hc = b.take<uint16_t>(s.op_planes * s.rows_pad * s.ld_h);
    l.row_top = b.take<uint32_t>(s.row_tops());
    if (c.loss) l.partial = b.take<float4>(s.slots * (s.keep ? s.rows : s.stat_rows));
    if (s.keep) l.ent_s = b.take<float>(s.rows_pad * K);
    if (s.dh_sum_rows) l.dh_sums = b.take<float>(s.dh_sum_rows * s.ld_acc);
    if (s.dw_sum_rows) l.dw_sums = b.take<float>(s.dw_sum_rows * s.ld_acc);
    if (s.dw_padded) l.dw_rows = b.take<uint8_t>(std::min(s.piece, s.V) * round_up(s.D * (s.f32 ? 4 : 2), 16));
    if (s.pack_w) l.wp = b.take<uint16_t>(s.op_planes * round_up(s.piece, kBK) * s.ld_h);
    if (s.grads) l.grad = b.take<uint16_t>(s.planes * s.rows * round_up(s.piece, 64));
    return l;
}

template <bool kF32>
int run(const Call& c, const Shape& s, const Layout& l, cudaStream_t stream) {
    const sw_linear_head& p = *c.plan;
    constexpr bool kBf16 = !kF32;
    const int esize = kF32 ? 4 : 2, terms = kF32 ? 3 : 1, sms = device_sms();
    const unsigned fill = (unsigned)(8 * sms);
    const int top_k = c.targets ? 1 : c.top_k;
    // rows of dim elements that the vector kernels can read
    auto whole_rows = [&](const void* x, int64_t sr, int64_t sc) {
        return sc == 1 && s.D % 8 == 0 && sr * esize % 16 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    };
    if (s.flags)
        SW_CUDA_TRY(launch_pdl(teacher_flags_kernel, dim3((unsigned)((s.T + 7) / 8)), dim3(256), 0, stream,
                               c.teacher_index, c.teacher_logits, s.T, c.top_k, s.V, l.flags),
                    "teacher rows");
    PrepareArgs pa;
    memset(&pa, 0, sizeof(pa));
    pa.targets = c.targets;
    pa.ignore_index = c.ignore_index;
    pa.index = c.teacher_index;
    pa.logits = c.teacher_logits;
    pa.flags = l.flags;
    pa.top_k = top_k;
    pa.inv_tau = c.scale;
    pa.T = s.T;
    pa.V = s.V;
    pa.rows_pad = (int)s.rows_pad;
    pa.entry_tiles = (int)((s.V + kEntryTile - 1) / kEntryTile);
    pa.upstream = c.upstream;
    pa.mean = p.reduction == SW_HEAD_MEAN;
    pa.factor = c.scale * c.factor;
    pa.lse = c.loss ? nullptr : c.lse;
    pa.row_map = l.row_map;
    pa.row_top = l.row_top;
    pa.row_tops = (int)s.row_tops();
    pa.ent_idx = l.ent_idx;
    pa.ent_p = l.ent_p;
    pa.entropy = l.entropy;
    pa.offs = l.offs;
    pa.coef = s.grads ? l.coef : nullptr;
    pa.norm = l.norm;
    pa.state = l.state;
    if (c.dh) {
        pa.dh_rows = s.rows;
        pa.dh_cols = s.D;
        pa.dh_k = std::min(s.piece, s.V);
    }
    pa.dh_shape = s.dh_shape;
    pa.sms = sms;
    pa.terms = terms;
    if (kBf16) {
        pa.h = static_cast<const uint16_t*>(c.h);
        pa.D = s.D;
        pa.sr = p.h_row;
        pa.sc = p.h_col;
        pa.vec = whole_rows(c.h, p.h_row, p.h_col);
        pa.hc = l.hc;
        pa.ld = s.ld_h;
        if (!pa.h) pa.h = l.hc;  // no rows: only zeros are written
    }
    // 8 rows a CTA for parallelism; 32 where every CTA's look at all T rows would show
    // Where there are few rows, several CTAs share the packing of 8 (2 column-major
    // rows of 2880 against 765 classes: 50 us with one CTA, 29 so).
    const int64_t blocks = s.rows_pad / 8, chunks = kBf16 ? (s.ld_h + 255) / 256 : 1;
    const unsigned shares = (unsigned)std::max<int64_t>(1, std::min<int64_t>(chunks, sms / blocks));
    if (s.T <= 16384)
        SW_CUDA_TRY(launch_pdl(prepare_kernel<8>, dim3((unsigned)blocks, shares), dim3(256), 0, stream, pa),
                    "linear head rows");
    else
        SW_CUDA_TRY(launch_pdl(prepare_kernel<32>, dim3((unsigned)(s.rows_pad / 32)), dim3(256), 0, stream, pa),
                    "linear head rows");
    auto job = [&](const void* x, int64_t rows, int64_t sr, int64_t sc, const int* map, int scale_of, uint16_t* dst,
                   int64_t rows_pad) {
        SplitJob j;
        memset(&j, 0, sizeof(j));
        j.src = x;
        j.rows = rows;
        j.cols = s.D;
        j.sr = sr;
        j.sc = sc;
        j.vec = whole_rows(x, sr, sc);
        j.row_map = map;
        j.scale_of = scale_of;
        j.dst = dst;
        j.ld = s.ld_h;
        j.rows_pad = rows_pad;
        j.parts = 1;
        const int64_t units = j.vec ? rows_pad * (s.D / 8) / 256 : (rows_pad + 31) / 32 * ((s.ld_h + 31) / 32);
        j.ctas = (unsigned)std::max<int64_t>(std::min<int64_t>(units, fill), 1);
        return j;
    };
    SplitJob none_job;
    memset(&none_job, 0, sizeof(none_job));
    auto split = [&](const SplitJob& j0, const SplitJob& j1) -> int {
        SW_CUDA_TRY(launch_pdl(split_kernel<kF32>, dim3(j0.ctas + j1.ctas), dim3(256), 0, stream, j0, j1, l.state),
                    "linear head operands");
        return SW_OK;
    };
    int rc;
    // the weights of columns [v0, v0 + n): in place, or packed into the workspace,
    // with zero rows up to whole K stages (a tail of G's zeros must not meet the
    // next plane); the first piece together with the states
    int64_t packed = -1;
    auto weight_job = [&](int64_t v0, int64_t n) {
        return job(static_cast<const uint8_t*>(c.w) + v0 * p.w_row * esize, n, p.w_row, p.w_col, nullptr, 1, l.wp,
                   round_up(n, kBK));
    };
    if (kF32) {
        SplitJob jh = job(c.h, s.T, p.h_row, p.h_col, l.row_map, 0, l.hc, s.rows_pad);
        const int64_t n = std::min(s.piece, s.V);
        SplitJob jw = weight_job(0, n), all = job(c.w, s.V, p.w_row, p.w_col, nullptr, 1, nullptr, s.V);
        jh.parts = s.h_parts;
        jh.row_top = l.row_top;
        jh.parts_in = jh.row_top + s.T;
        all.parts = s.w_parts;
        all.row_top = l.row_top + s.measured(s.T, s.h_parts);
        all.parts_in = all.row_top + s.V;
        SW_CUDA_TRY(launch_pdl(amax_kernel, dim3(jh.ctas + all.ctas), dim3(256), 0, stream, jh, all, l.state),
                    "linear head scales");
        if ((rc = split(jh, jw)) != SW_OK) return rc;
        packed = 0;
    }
    const Plane dense{kBK, 0, 0};
    // rows [r0, r0 + n) of the gathered states
    auto states = [&](int64_t r0, int64_t n) {
        return Operand{l.hc + r0 * s.ld_h, (s.op_planes - 1) * s.rows_pad + n, s.D, s.ld_h, Plane{kBK, 0, (int)s.rows_pad}};
    };
    const int64_t ld_grad = s.planes * round_up(s.piece, 64);

    GemmArgs g;
    memset(&g, 0, sizeof(g));
    g.state = l.state;
    g.logit_scale = c.scale;
    g.ent_p = l.ent_p;
    g.ent_k = top_k;
    g.slots = (int)s.slots;
    g.slot_shift = s.slot_shift;
    g.tile_n = s.tile_n;
    g.rows_pad = (int)s.rows_pad;
    const Target grad_out{l.grad, s.rows, ld_grad, ld_grad, false}, none{nullptr, 0, 0, 0, false};

    auto weights = [&](int64_t v0, int64_t n, Operand* out) -> int {
        if (!s.pack_w) {
            const uint8_t* at = static_cast<const uint8_t*>(c.w) + v0 * p.w_row * esize;
            *out = Operand{reinterpret_cast<const uint16_t*>(at), n, s.D, p.w_row, dense};
            return SW_OK;
        }
        const int64_t rows = round_up(n, kBK);
        if (packed != v0 && (rc = split(weight_job(v0, n), none_job)) != SW_OK) return rc;
        packed = v0;
        *out = Operand{l.wp, s.op_planes * rows, s.D, s.ld_h, Plane{kBK, 0, (int)rows}};
        return SW_OK;
    };
    // logits of compact rows [r0, r0 + n) and columns [v0, v0 + nv)
    auto logits = [&](int64_t r0, int64_t n, int64_t v0, int64_t nv) {
        GemmArgs a = g;
        a.problems = 1;
        a.p[0].M = (int)n;
        a.p[0].N = (int)nv;
        a.p[0].K = (int)s.D;
        a.p[0].count_is = kCountM;
        a.p[0].splits = 1;
        a.p[0].scale_a = kF32 ? 0 : -1;
        a.p[0].scale_b = kF32 ? 1 : -1;
        a.row0 = (int)r0;
        a.v0 = v0;
        a.ent_idx = l.ent_idx + r0 * g.ent_k;
        a.ent_p = l.ent_p ? l.ent_p + r0 * g.ent_k : nullptr;
        a.offs = l.offs ? l.offs + r0 : nullptr;
        a.partial = l.partial;
        // what the row subtracts: the kept lse of the logits, or the largest z and the sum's logarithm
        a.norm = l.norm + r0;
        a.to_ref = c.loss ? 1.0f : c.scale;
        a.to_log2 = c.loss ? c.scale * kLog2e : kLog2e;
        a.factor_rest = c.loss ? 0.0f : float((double(c.scale) * kLog2e - double(c.scale * kLog2e)) / c.scale);
        a.coef = l.coef + r0;
        return a;
    };
    // the loss of compact rows [r0, r0 + n), and with `grad` their logits' gradient
    auto losses = [&](int64_t r0, int64_t n, bool grad) -> int {
        LossArgs a;
        memset(&a, 0, sizeof(a));
        a.partial = l.partial;
        a.slots = (int)s.slots;
        a.slot_shift = s.slot_shift;
        a.row0 = (int)r0;
        a.rows = (int)n;
        a.all_rows = (int)std::max<int64_t>(s.T, 1);
        a.state = l.state;
        a.row_map = l.row_map;
        a.targets = c.targets;
        a.ignore_index = c.ignore_index;
        a.entropy = l.entropy;
        a.factor = c.factor;
        a.row_loss = l.row_loss;
        a.logit_scale = c.scale;
        a.norm = l.norm;
        a.loss = c.loss;
        a.mean = p.reduction == SW_HEAD_MEAN;
        a.lse = c.lse;
        int64_t segs = 1;
        if (grad) {
            // a CTA takes a whole row, or where rows are few a part of one of at
            // least 2048 columns
            segs = std::max<int64_t>(1, std::min<int64_t>((s.V + 2047) / 2048, 4 * sms / std::max<int64_t>(n, 1)));
            a.grad = l.grad;
            a.ld_grad = ld_grad;
            a.V = s.V;
            a.seg = round_up((s.V + segs - 1) / segs, 512);
            segs = (s.V + a.seg - 1) / a.seg;
            a.coef = l.coef;
            a.ent_idx = l.ent_idx;
            a.ent_p = l.ent_p;
            a.ent_s = l.ent_s;
            a.ent_k = top_k;
        }
        SW_CUDA_TRY(launch_pdl(loss_kernel<kF32>, dim3((unsigned)std::max<int64_t>(n, 1), (unsigned)segs), dim3(256), 0,
                               stream, a),
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
            PlaceArgs sa;
            memset(&sa, 0, sizeof(sa));
            sa.sums = sums;
            sa.ld = s.ld_acc;
            sa.splits = splits;
            sa.tile_m = shape_rows(shape);
            sa.workers = shape_workers(shape, sms);
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
            const int64_t spans = (s.D + 1023) / 1024, per = rows * spans < 8 * sms ? 1 : 4;
            const int64_t share = std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, fill / spans));
            const dim3 grid((unsigned)spans, (unsigned)share);
            SW_CUDA_TRY(per == 1 ? launch_pdl(place_kernel<kF32, 1>, grid, dim3(256), 0, stream, sa)
                                 : launch_pdl(place_kernel<kF32, 4>, grid, dim3(256), 0, stream, sa),
                        "linear head sums");
            return SW_OK;
        };
        Tensors t[2];
        const int64_t ld_rows = round_up(s.D * esize, 16) / esize;
        uint8_t* dw = c.dw ? static_cast<uint8_t*>(c.dw) + v0 * p.dw_row * esize : nullptr;
        if (c.dh && n > 0) {
            Problem& q = a.p[a.problems];
            q.M = (int)n;
            q.N = (int)s.D;
            q.K = (int)nv;
            q.count_is = kCountM;
            q.scale_a = kF32 ? 2 : -1;
            q.scale_b = kF32 ? 1 : -1;
            q.splits = 0;
            q.sums = 1;
            q.first = first_v;
            t[a.problems++] = Tensors{gr, w, Target{l.dh_sums, s.dh_sum_rows, s.ld_acc, s.ld_acc, true}};
        }
        if (dw) {
            Problem& q = a.p[a.problems];
            q.M = (int)nv;
            q.N = (int)s.D;
            q.K = (int)n;
            q.count_is = kCountK;
            q.a_mn = 1;
            q.scale_a = kF32 ? 2 : -1;
            q.scale_b = kF32 ? 0 : -1;
            q.splits = s.dw_splits;
            q.sums = s.dw_sum_rows > 0;
            q.first = first_r;
            Target out{dw, nv, s.D, p.dw_row, kF32};
            // (a map whose rows end inside 16 bytes would be written past them: whole ones here)
            if (s.dw_padded) out = Target{l.dw_rows, nv, ld_rows, ld_rows, kF32};
            if (q.sums) out = Target{l.dw_sums, s.dw_sum_rows, s.ld_acc, s.ld_acc, true};
            const Operand st = states(r0, round_up(std::max<int64_t>(n, 1), kBM));
            t[a.problems++] = Tensors{gr, st, out};
        }
        int rc = SW_OK;
        if (a.problems == 2 && s.together) {
            a.alternate = 1;
            rc = gemm<kBf16, kEpiOut, kBoth>(t, a, kSingle, stream);
        } else {
            const bool two = a.problems == 2;
            a.problems = 1;
            if (c.dh && n > 0) rc = gemm<kBf16, kEpiOut, kKMajor>(t, a, s.dh_shape, stream);
            if (rc == SW_OK && dw) {
                if (two) {
                    t[0] = t[1];
                    a.p[0] = a.p[1];
                }
                rc = gemm<kBf16, kEpiOut, kMnMajor>(t, a, s.dw_shape, stream);
            }
        }
        if (rc == SW_OK && c.dh && n > 0 && last_v)
            rc = finish(l.dh_sums, 0, s.dh_shape, n, true, l.row_map + r0, c.dh, p.dh_row, p.dh_col);
        if (rc == SW_OK && s.dw_sum_rows && last_r)
            rc = finish(l.dw_sums, s.dw_splits, s.dw_shape, nv, false, nullptr, dw, p.dw_row, p.dw_col);
        if (rc == SW_OK && s.dw_padded) {
            using E = typename std::conditional<kF32, float, uint16_t>::type;
            SW_CUDA_TRY(launch_pdl(unpad_kernel<E>, dim3((unsigned)std::min<int64_t>((nv * s.D + 2047) / 2048, fill)),
                                   dim3(256), 0, stream, static_cast<const E*>(l.dw_rows), ld_rows, nv, s.D,
                                   reinterpret_cast<E*>(dw), p.dw_row, p.dw_col),
                        "linear head dw");
        }
        return rc;
    };
    if (s.keep) {
        Operand w;
        if ((rc = weights(0, s.V, &w)) != SW_OK) return rc;
        for (int64_t r0 = 0; r0 == 0 || r0 < s.T; r0 += s.rows) {
            const int64_t n = std::min(s.rows, s.T - r0);
            GemmArgs a = logits(r0, n, 0, s.V);
            a.keep = 1;
            a.ent_s = l.ent_s + r0 * g.ent_k;
            const Tensors t{states(r0, round_up(std::max<int64_t>(n, 1), kBM)), w, grad_out};
            if ((rc = gemm<kBf16, kEpiLse, kKMajor>(&t, a, s.logits_shape, stream)) != SW_OK) return rc;
            if ((rc = losses(r0, n, true)) != SW_OK) return rc;
            if ((rc = gradients(r0, n, 0, s.V, w, true, true, r0 == 0, r0 + s.rows >= s.T)) != SW_OK) return rc;
        }
        return SW_OK;
    }
    if (c.loss) {
        const int64_t step = s.pack_w ? s.piece : s.V;
        for (int64_t r0 = 0; r0 == 0 || r0 < s.T; r0 += s.stat_rows) {
            const int64_t nr = std::min(s.stat_rows, s.T - r0);
            for (int64_t v0 = 0; v0 < s.V; v0 += step) {
                const int64_t n = std::min(step, s.V - v0);
                Operand w;
                if ((rc = weights(v0, n, &w)) != SW_OK) return rc;
                GemmArgs a = logits(r0, nr, v0, n);
                const Tensors t{states(r0, round_up(std::max<int64_t>(nr, 1), kBM)), w, none};
                if ((rc = gemm<kBf16, kEpiLse, kKMajor>(&t, a, s.logits_shape, stream)) != SW_OK) return rc;
            }
            if ((rc = losses(r0, nr, false)) != SW_OK) return rc;
        }
    }
    if (!s.grads) return SW_OK;
    for (int64_t v0 = 0; v0 < s.V; v0 += s.piece) {
        const int64_t n = std::min(s.piece, s.V - v0);
        Operand w;
        if ((rc = weights(v0, n, &w)) != SW_OK) return rc;
        GemmArgs a = logits(0, s.T, v0, n);
        const Tensors t{states(0, s.rows_pad), w, grad_out};
        const bool cut = kBf16 && s.D > int64_t(kBK) * chunk_stages(true, kEpiGradCut, a);
        rc = cut ? gemm<kBf16, kBf16 ? kEpiGradCut : kEpiGrad, kKMajor>(&t, a, s.logits_shape, stream)
                 : gemm<kBf16, kEpiGrad, kKMajor>(&t, a, s.logits_shape, stream);
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
    // i sr = j sc first for i = sc / g, j = sr / g
    const int64_t g = std::gcd(sr, sc);
    return sc / g >= rows || sr / g >= cols;
}

// A call's plan: `keep` with the exponentials of `rows` compact rows at a time, or
// the logits' gradient of `piece` columns of the vocabulary, and the statistics of
// a loss alone of `stat_rows` rows at a time.
Shape make_plan(const Call& c, bool keep, int64_t rows, int64_t piece, int64_t stat_rows) {
    const sw_linear_head* p = c.plan;
    const int64_t T = p->tokens, D = p->dim, V = p->vocab;
    const bool grads = c.dh || c.dw;
    Shape s;
    s.T = T;
    s.D = D;
    s.V = V;
    s.f32 = p->dtype == SW_HEAD_F32;
    s.planes = s.f32 ? 2 : 1;
    s.op_planes = s.f32 ? 3 : 1;
    // 32 rows a CTA, and where that leaves SMs idle parts of at least 64 columns
    auto parts = [&](int64_t rows, int64_t sr, int64_t sc) {
        if (!s.f32 || sr != 1 || sc == 1) return 1;
        const int64_t items = (rows + 31) / 32, want = 4 * device_sms();
        return (int)std::max<int64_t>(1, items * 2 > want ? 1 : std::min((D + 63) / 64, want / std::max<int64_t>(items, 1)));
    };
    s.h_parts = parts(T, p->h_row, p->h_col);
    s.w_parts = parts(V, p->w_row, p->w_col);
    s.rows_pad = std::max<int64_t>(round_up(T, kBM), kBM);
    s.ld_h = round_up(D, 8);
    s.flags = !c.targets && T * c.top_k > kInlineFlags;
    s.grads = grads;
    s.ld_acc = round_up(D, 4);
    // weights are read in place when TMA can: bf16, unit stride, 16-byte rows
    s.pack_w = s.f32 || p->w_col != 1 || p->w_row % 8 != 0 || p->w_row < D ||
               (reinterpret_cast<uintptr_t>(c.w) & 15) != 0;
    const int terms = s.f32 ? 3 : 1;
    s.keep = keep;
    s.rows = rows;
    s.piece = piece;
    s.stat_rows = stat_rows;
    const int64_t n = std::min(s.rows, T), nv = std::min(s.piece, V), nl = grads ? n : std::min(stat_rows, T);
    // (a pair's second half would have no row of a single row tile: 21 x 18689 at dim
    // 2496 scored in 45 us by pairs, in 32 by single CTAs)
    s.logits_shape = nl <= kBM || choose_parts(nl, nv, D, terms, kSingle, false).us <
                              0.97f * choose_parts(nl, nv, D, terms, kPair2, false).us
                         ? kSingle
                         : kPair2;
    // Where 256-column tiles would leave SMs idle, and 128 or 64 columns still make one
    // wave, those spread the weights over more of them: the loss of one token over 16000
    // classes at dim 4096 44.1 us at 256 columns, 41.0 at 128, over 8000 40.2, 34.6 at 64;
    // Float32 33 x 1021 at dim 257 with gradients 53.3, 47.6 at 64.
    s.tile_n = kBN;
    if (s.logits_shape == kSingle)
        for (const int t : {128, 64})
            if ((nl + kBM - 1) / kBM * ((nv + t - 1) / t) <= device_sms()) s.tile_n = t;
    s.slot_shift = s.tile_n == 64 ? 6 : 7;
    s.slots = (V + s.tile_n - 1) / s.tile_n * (s.tile_n >> s.slot_shift);
    // dw is written at once through TMA where that can describe it (rows that end
    // inside 16 bytes would be written past their end).
    const int64_t es = s.f32 ? 4 : 2;
    const bool direct = p->dw_col == 1 && p->dw_row * es % 16 == 0 && D * es % 16 == 0 && p->dw_row >= D &&
                        (reinterpret_cast<uintptr_t>(c.dw) & 15) == 0;
    const bool one_part = s.rows >= T;  // nothing to add to what is written
    const float sum_us = one_part ? float(nv) * float(D) * float(8 + es) / 6.0e6f : 0.0f;
    s.together = c.dh && c.dw && n <= kBM;
    s.dh_shape = s.dw_shape = kSingle;
    s.dw_splits = 1;
    float dh_us = 1e30f, dw_us = 1e30f;
    for (int shape = s.together ? kSingle : s.f32 ? kPair2 : kTall; grads && shape >= kSingle; --shape) {
        const Spread dh = choose_parts(n, D, nv, terms, shape, true);
        const Spread dw = choose_parts(nv, D, n, terms, shape, true, sum_us);
        if (dh.us < dh_us * 0.97f) {
            dh_us = dh.us;
            s.dh_shape = shape;
        }
        if (dw.us < dw_us * 0.97f) {
            dw_us = dw.us;
            s.dw_shape = shape;
            s.dw_splits = dw.splits;
        }
    }
    s.dh_sum_rows = c.dh && T > 0 ? sum_rows(n, D, most_parts(nv), s.dh_shape, device_sms()) : 0;
    s.dw_sum_rows = c.dw && (!one_part || s.dw_splits > 1) ? sum_rows(nv, D, s.dw_splits, s.dw_shape, device_sms()) : 0;
    s.dw_padded = c.dw && !s.dw_sum_rows && !direct;
    return s;
}

int64_t scratch_bytes(const Call& c, const Shape& s) {
    Bump measure{nullptr, 0};
    lay_out(measure, c, s);
    return measure.used;
}

// The plan that does least within the workspace limit.  One call for the loss and
// the gradients keeps the logits' exponentials of all rows, or of as many as fit,
// 1024 (or all) at least, beside the fp32 sums of dw that blocks of rows need (6
// T V D operations and one more pass over them).  From a kept lse, or where that
// does not fit, the logits are computed again (8 T V D), in pieces of the
// vocabulary as wide as fit, in whole 256-column tiles.  The least there is - one
// such piece, and the statistics of 1024 rows - is taken even if it does not fit.
Shape choose_plan(const Call& c) {
    const sw_linear_head* p = c.plan;
    const bool grads = c.dh || c.dw;
    const int64_t limit = p->workspace_limit > 0 ? p->workspace_limit : kDefaultWorkspace;
    const int64_t all = std::max<int64_t>(round_up(p->tokens, kBM), kBM), fewest = std::min<int64_t>(all, 1024);
    const int64_t whole = round_up(p->vocab, 256);
    auto bytes = [&](const Shape& s) { return scratch_bytes(c, s); };
    // the largest multiple of `unit` from `least` to `most` whose plan fits; the bytes grow with it
    auto largest = [&](int64_t least, int64_t most, int64_t unit, auto&& plan) {
        int64_t lo = least / unit, hi = (most + unit - 1) / unit;
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) / 2;
            if (bytes(plan(std::min(mid * unit, most))) <= limit) lo = mid;
            else hi = mid - 1;
        }
        return std::min(lo * unit, most);
    };
    if (c.loss && grads) {
        auto kept = [&](int64_t rows) { return make_plan(c, true, rows, whole, rows); };
        const Shape s = kept(all);
        if (bytes(s) <= limit) return s;
        if (fewest < all && bytes(kept(fewest)) <= limit) {
            const int64_t rows = largest(fewest, all - kBM, kBM, kept), blocks = (all + rows - 1) / rows;
            const Shape even = kept(round_up((all + blocks - 1) / blocks, kBM));
            return bytes(even) <= limit ? even : kept(rows);
        }
    }
    auto again = [&](int64_t piece, int64_t stat_rows) { return make_plan(c, false, all, piece, stat_rows); };
    Shape s = again(whole, all);
    if (bytes(s) <= limit) return s;
    // packed weights are packed once for all rows' statistics, so in pieces these are not blocked
    if (!grads && (!s.pack_w || bytes(again(whole, fewest)) <= limit))
        return again(whole, largest(fewest, all, kBM, [&](int64_t rows) { return again(whole, rows); }));
    const int64_t stats = s.pack_w ? all : fewest;
    const int64_t piece = largest(256, whole, 256, [&](int64_t columns) { return again(columns, stats); });
    if (s.pack_w || !c.loss) return again(piece, stats);
    return again(piece, largest(fewest, all, kBM, [&](int64_t rows) { return again(piece, rows); }));
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

    const Shape s = choose_plan(c);
    const int64_t bytes = scratch_bytes(c, s);
    void* ws = nullptr;
    int dev = 0;
    SW_CUDA_TRY(cudaGetDevice(&dev), "cudaGetDevice");
    const int pooled = keep_pool_memory(dev);
    if (pooled != SW_OK) return pooled;
    cudaError_t err = cudaMallocAsync(&ws, (size_t)bytes, stream);
    if (err == cudaErrorMemoryAllocation) {
        cudaGetLastError();
        return fail(SW_ERR_NOMEM, "%s: out of device memory for %lld bytes of workspace", name,
                    (long long)bytes);
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
