// Entry points of the gated feed-forward block (kla_mlp.cuh): argument checks, tensor maps, tile choice, launches.
#include <algorithm>
#include <atomic>
#include <mutex>

#include "../../include/kla_b200.h"
#include "kla_entry.h"
#include "kla_launch.cuh"
#include "kla_mlp.cuh"

namespace {

using namespace kla;

bool aligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
bool rows_of_16(const void *p, int64_t stride) { return aligned(p, 16) && stride % 8 == 0; }
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to; }

// A [halves][outer][inner] bfloat16 tensor of boxes box_inner (64, or 32 of a warp's stage) x box_outer, swizzled by a row of the box.
int make_map(CUtensorMap *tm, const void *p, int64_t inner, int64_t outer, int64_t stride, int64_t halves, int64_t half_stride, int box_outer,
             int box_inner = 64) {
    entry::EncodeTiledFn enc = entry::encode_tiled_fn();
    if (enc == nullptr) return KLA_B200_EUNSUPPORTED;
    const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)halves};
    const cuuint64_t strides[2] = {(cuuint64_t)stride * 2, (cuuint64_t)(halves > 1 ? half_stride : stride * outer) * 2};
    const cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1}, ones[3] = {1, 1, 1};
    const CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           box_inner == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? KLA_B200_OK : KLA_B200_EINVAL;
}

// An operand in memory: `rows` of the product by the summed axis. adjacent_rows: the rows are the adjacent axis.
struct Operand {
    const void *p;
    int64_t stride, half_stride;
    bool adjacent_rows;
    int halves;
};
struct Product {
    Operand a, b;
    int64_t M, N, K;  // N, K of one half where halves are
    int mode;
    bool gated() const { return b.halves == kHalvesBoth; }
};
struct Plan {
    int BN, CG, tiles_m, tiles_n, splits;
};

// Columns of a tile, CTAs sharing it and shares of the summed axis: the least time (us) by what was measured on B200. A CTA spends
// `block` on a 64-wide block of its tile with the GPU full (two CTAs with 256 columns 0.40, one 0.42; K=4096 N=1024 of 18944 rows) and
// `fixed` on a launch, its first loads and its last epilogue (one block of 64 rows: pairs of CTAs 8.3, one CTA 6.2 to 7.7). Partial
// sums are written, and read again by a kernel more, 2.5 us: 64 rows of 768 with H = 2048 forward 20.5 us whole, 16.4 split, 512 rows
// 20.6 and 20.7, 300 rows of 1000 with H = 3000 30.8 and 25.1.
Plan plan(const Product &p, bool may_split, int sms) {
    const int64_t blocks = up(p.K, kMlpBK) * (p.a.halves == kHalvesSummed ? 2 : 1);
    constexpr struct { int bn; double block[2], fixed[2]; } kinds[] = {
        {256, {0.42, 0.40}, {7.5, 8.3}}, {192, {0.34, 0.32}, {6.7, 8.3}}, {128, {0.24, 0.25}, {6.2, 8.3}}, {64, {0.20, 0.215}, {6.2, 8.3}}};
    Plan best{};
    double least = 0.0;
    for (const int cg : {2, 1})
        for (const auto &kind : kinds) {
            const int bn = kind.bn;
            if (p.gated() && bn == 64) continue;
            const int64_t tm = up(p.M, kMlpBM * cg) * (p.a.halves == kHalvesRows ? 2 : 1);
            const int64_t tn = up(p.N, p.gated() ? bn / 2 : bn), tiles = tm * tn;
            // shares of the summed axis up to four rounds of CTAs
            const int64_t most = may_split ? std::min<int64_t>({32, blocks, 1 + 4 * sms / (tiles * cg)}) : 1;
            for (int s = 1; s <= most; ++s) {
                const double sums = s > 1 ? 2.5 + 8e-6 * s * (double)tm * tn * kMlpBM * cg * bn / 4.0 : 0.0;
                const double thin = p.gated() ? (bn == 128 ? 1.2 : bn == 192 ? 1.1 : 1.0) : 1.0;  // fewer than 128 columns of h leave warps of the epilogue idle
                const double t = (double)up(tiles * s, sms / cg) * up(blocks, s) * kind.block[cg - 1] * thin + kind.fixed[cg - 1] + sums;
                if (best.BN == 0 || t < least) { best = Plan{bn, cg, (int)tm, (int)tn, s}; least = t; }
            }
        }
    return best;
}

int fill(MlpParams *prm, const Product &p, const Plan &pl) {
    *prm = MlpParams{};
    // tensor maps are made by the driver for the thread's context, which a new thread (autograd's, or a caller's) has only
    // once the runtime has bound it
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaSetDevice(dev);
    if (e != cudaSuccess) return entry::cuda_fail(e);
    const int64_t mh = p.a.halves == kHalvesNone ? 1 : 2, nh = p.b.halves == kHalvesNone ? 1 : 2;
    int rc = p.a.adjacent_rows ? make_map(&prm->map_a, p.a.p, p.M, p.K, p.a.stride, mh, p.a.half_stride, kMlpBK)
                               : make_map(&prm->map_a, p.a.p, p.K, p.M, p.a.stride, mh, p.a.half_stride, kMlpBM);
    if (rc) return rc;
    rc = p.b.adjacent_rows ? make_map(&prm->map_b, p.b.p, p.N, p.K, p.b.stride, nh, p.b.half_stride, kMlpBK)
                           : make_map(&prm->map_b, p.b.p, p.K, p.N, p.b.stride, nh, p.b.half_stride, p.gated() ? pl.BN / 2 : pl.BN / pl.CG);
    if (rc) return rc;
    prm->a = MlpOperand{p.a.adjacent_rows, p.a.halves};
    prm->b = MlpOperand{p.b.adjacent_rows, p.b.halves};
    prm->M = (int)p.M; prm->N = (int)p.N; prm->K = (int)p.K;
    prm->BN = pl.BN; prm->tiles_m = pl.tiles_m; prm->tiles_n = pl.tiles_n; prm->splits = pl.splits;
    prm->stages = std::min(kMlpMaxStages, kMlpRingBytes / mlp_block_bytes(pl.BN, pl.CG, p.b.adjacent_rows));
    prm->blocks_stretch = (int)up(p.K, kMlpBK);
    prm->blocks_k = prm->blocks_stretch * (p.a.halves == kHalvesSummed ? 2 : 1);
    return entry::wait_ctl(&prm->wait);
}

// A launch that may begin before the kernel in front of it has ended: the kernels wait (grid_dep_wait) before they touch memory.
template <typename Params>
int launch_behind(void (*kern)(Params), dim3 grid, unsigned threads, size_t smem, int cluster, cudaStream_t st, const Params &prm) {
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, prm);
    if (e != cudaSuccess) return entry::cuda_fail(e);
    entry::count_launch();
    return KLA_B200_OK;
}

// CTA pairs that can be resident at once: SMs without a partner in their cluster of SMs take none.
int resident_pairs() {
    static std::mutex mu;
    static int pairs[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return device_sms() / 2;
    std::lock_guard<std::mutex> lock(mu);
    if (pairs[dev] == 0) {
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)device_sms() / 2 * 2);
        cfg.blockDim = dim3(kMlpThreads);
        cfg.dynamicSmemBytes = kMlpSmem;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kla_mlp_kernel<kMlpPlain, 2>, &cfg) != cudaSuccess || n < 1) {
            cudaGetLastError();
            return device_sms() / 2;
        }
        pairs[dev] = n;
    }
    return pairs[dev];
}

// The kernel may use its shared memory; asked for once per device.
template <int MODE, int CG>
cudaError_t allow_smem() {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && done.load() >> dev & 1)) return e;
    e = cudaFuncSetAttribute(kla_mlp_kernel<MODE, CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMlpSmem);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev);
    return e;
}

template <int MODE, int CG>
int launch_as(const MlpParams &prm, cudaStream_t st) {
    cudaError_t e = allow_smem<MODE, CG>();
    if (e == cudaSuccess && CG == 2) e = allow_smem<kMlpPlain, 2>();  // (resident_pairs asks about that kernel)
    if (e != cudaSuccess) return entry::cuda_fail(e);
    const int64_t tiles = (int64_t)prm.tiles_m * prm.tiles_n * prm.splits;
    if (tiles > 0x3fffffffll) return KLA_B200_EUNSUPPORTED;
    const int64_t most = CG == 2 ? resident_pairs() : device_sms();
    return launch_behind(kla_mlp_kernel<MODE, CG>, dim3((unsigned)(tiles < most ? tiles : most) * CG), kMlpThreads, kMlpSmem, CG, st, prm);
}
template <int MODE>
int launch(const MlpParams &prm, const Plan &pl, cudaStream_t st) {
    return pl.CG == 2 ? launch_as<MODE, 2>(prm, st) : launch_as<MODE, 1>(prm, st);
}

Product product(const Operand &a, const Operand &b, int64_t M, int64_t N, int64_t K, int mode) { return Product{a, b, M, N, K, mode}; }
Operand plain(const void *p, int64_t stride, bool adjacent_rows = false) { return Operand{p, stride, 0, adjacent_rows, kHalvesNone}; }

Product product_gate_up(const kla_b200_mlp_args &a) {
    return product(plain(a.x, a.x_stride), Operand{a.w12, a.w12_stride, a.w12_stride * a.H, false, kHalvesBoth}, a.rows, a.H, a.d, kMlpGated);
}
Product product_down(const kla_b200_mlp_args &a) { return product(plain(a.h, a.h_stride), plain(a.w3, a.w3_stride), a.rows, a.out, a.H, kMlpPlain); }
Product product_dgu(const kla_b200_mlp_args &a) { return product(plain(a.dy, a.dy_stride), plain(a.w3, a.w3_stride, true), a.rows, a.H, a.out, kMlpGrad); }
Product product_dx(const kla_b200_mlp_args &a) {
    return product(Operand{a.dgu, a.gu_stride, a.gu_stride / 2, false, kHalvesSummed},
                   Operand{a.w12, a.w12_stride, a.w12_stride * a.H, true, kHalvesSummed}, a.rows, a.d, a.H, kMlpPlain);
}
Product product_dw3(const kla_b200_mlp_args &a) { return product(plain(a.dy, a.dy_stride, true), plain(a.h, a.h_stride, true), a.out, a.H, a.rows, kMlpPartial); }
Product product_dw12(const kla_b200_mlp_args &a) {
    return product(Operand{a.dgu, a.gu_stride, a.gu_stride / 2, true, kHalvesRows}, plain(a.x, a.x_stride, true), a.H, a.d, a.rows, kMlpPartial);
}

int64_t product_rows(const Product &p) { return p.M * (p.a.halves == kHalvesRows ? 2 : 1); }
int64_t partial_words(const Product &p, int sms) {
    const int splits = plan(p, true, sms).splits;
    return splits > 1 ? splits * product_rows(p) * up(p.N, 4) * 4 : 0;
}
// rows of a stretch of the row sums: at least eight a warp, and no more than 1024 stretches
int64_t sum_rows(int64_t rows) { return std::max<int64_t>(64, up(rows, 1024 * 8) * 8); }

// The working memory of a backward, in words: partial sums of dW3, dW12 and dx, of db3 and db12.
struct Work {
    int64_t w12, dx, b3, b12, all;  // where they begin (dW3's at 0)
};
Work work_of(const kla_b200_mlp_args &a, int sms) {
    const int64_t stretches = up(a.rows, sum_rows(a.rows));
    Work w;
    w.w12 = partial_words(product_dw3(a), sms);
    w.dx = w.w12 + partial_words(product_dw12(a), sms);
    w.b3 = w.dx + partial_words(product_dx(a), sms);
    w.b12 = w.b3 + stretches * a.out;
    w.all = w.b12 + stretches * 2 * a.H;
    return w;
}

// What a product without activation is stored to, with what is added to it. half: elements to the second half of the rows
struct Result {
    void *out;
    int64_t stride, half;
    const void *bias, *side;
    int64_t side_stride;
};
// In one go, or (may_split) partial sums of shares of the summed axis, to be added by the end's kernel.
int launch_plain(const Product &p, const Result &r, bool may_split, float *work, MlpReduce *end, cudaStream_t st) {
    const Plan pl = plan(p, may_split, device_sms());
    MlpParams prm;
    if (const int rc = fill(&prm, p, pl)) return rc;
    if (pl.splits == 1) {
        prm.out = static_cast<__nv_bfloat16 *>(r.out); prm.out_stride = r.stride; prm.out_half = r.half; prm.out_vec = rows_of_16(r.out, r.stride);
        prm.bias = static_cast<const __nv_bfloat16 *>(r.bias);
        prm.side = static_cast<const __nv_bfloat16 *>(r.side); prm.side_stride = r.side_stride; prm.side_vec = rows_of_16(r.side, r.side_stride);
        return launch<kMlpPlain>(prm, pl, st);
    }
    prm.partial = work;
    prm.partial_stride = up(p.N, 4) * 4;
    prm.partial_rows = product_rows(p);  // (halves of rows: the second's follow the first's in `out` too)
    *end = MlpReduce{work, prm.partial_rows * prm.partial_stride, prm.partial_stride, pl.splits, (int)prm.partial_rows, (int)p.N,
                     (int)up(prm.partial_rows * up(p.N, 4), 256), static_cast<__nv_bfloat16 *>(r.out), r.stride, aligned(r.out, 8) && r.stride % 4 == 0,
                     static_cast<const __nv_bfloat16 *>(r.bias), static_cast<const __nv_bfloat16 *>(r.side), r.side_stride};
    return launch<kMlpPartial>(prm, pl, st);
}
Result weight(void *out, const Product &p) { return Result{out, p.N, p.M * p.N, nullptr, nullptr, 0}; }

// The kernel that adds what is left to be added; of[].blocks: of each alone.
int launch_end(MlpEndParams *end, cudaStream_t st) {
    for (int i = 1; i < kMlpSums; ++i) end->of[i].blocks += end->of[i - 1].blocks;
    end->bias_blocks = end->of[kMlpSums - 1].blocks + (int)up(end->bias[0].total, 32);
    const int64_t blocks = end->bias_blocks + up(end->bias[1].total, 32);
    return blocks > 0 ? launch_behind(kla_mlp_end_kernel, dim3((unsigned)blocks), 256, 0, 1, st, *end) : KLA_B200_OK;
}

MlpSum sum_of(const void *x, int64_t stride, int64_t cols, int64_t half_gap, int halves, float *work, void *out) {
    const int half_blocks = (int)up(cols, kMlpSumCols);
    return MlpSum{static_cast<const __nv_bfloat16 *>(x), stride, half_gap, (int)cols, half_blocks, halves * half_blocks, (int)(halves * cols), work,
                  static_cast<__nv_bfloat16 *>(out)};
}

int check_sizes(const kla_b200_mlp_args *a) {
    if (a == nullptr || a->rows < 0 || a->d <= 0 || a->H <= 0 || a->out <= 0) return KLA_B200_EINVAL;
    if (a->activation < KLA_B200_ACT_SILU || a->activation > KLA_B200_ACT_NONE) return KLA_B200_EINVAL;
    if (a->rows > (1 << 30) || a->d > (1 << 24) || a->H > (1 << 24) || a->out > (1 << 24)) return KLA_B200_EUNSUPPORTED;
    return KLA_B200_OK;
}
// an operand of the tensor cores: rows of `width` elements, 16 bytes at a time
int check_operand(const void *p, int64_t stride, int64_t width) {
    if (p == nullptr || stride < width) return KLA_B200_EINVAL;
    return rows_of_16(p, stride) ? KLA_B200_OK : KLA_B200_EALIGN;
}
int check_plain(const void *p, int64_t stride, int64_t width) {
    if (p == nullptr || stride < width) return KLA_B200_EINVAL;
    return aligned(p, 2) ? KLA_B200_OK : KLA_B200_EALIGN;
}

}  // namespace

extern "C" {

int kla_b200_mlp_fwd(const kla_b200_mlp_args *a, void *stream) {
    int rc = check_sizes(a);
    if (rc) return rc;
    if (a->rows == 0) return KLA_B200_OK;
    if ((rc = check_operand(a->x, a->x_stride, a->d)) || (rc = check_operand(a->w12, a->w12_stride, a->d)) || (rc = check_operand(a->w3, a->w3_stride, a->H)) ||
        (rc = check_operand(a->h, a->h_stride, a->H)) || (rc = check_plain(a->y, a->y_stride, a->out)))
        return rc;
    if (a->gu != nullptr && (a->gu_stride % 16 || (rc = check_operand(a->gu, a->gu_stride, 2 * a->H)))) return rc ? rc : KLA_B200_EALIGN;
    if (a->residual != nullptr && (rc = check_plain(a->residual, a->residual_stride, a->out))) return rc;
    if (!aligned(a->b12, 2) || !aligned(a->b3, 2) || !aligned(a->work, 16)) return KLA_B200_EALIGN;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int sms = device_sms();
    MlpParams prm;
    const Product first = product_gate_up(*a), second = product_down(*a);
    const Plan pl = plan(first, false, sms);
    if ((rc = fill(&prm, first, pl))) return rc;
    prm.act = a->activation;
    prm.bias = static_cast<const __nv_bfloat16 *>(a->b12);
    if ((rc = make_map(&prm.map_out, a->h, a->H, a->rows, a->h_stride, 1, 0, 32, 32))) return rc;
    prm.keeps = a->gu != nullptr;
    if (prm.keeps && (rc = make_map(&prm.map_kept, a->gu, a->H, a->rows, a->gu_stride, 2, a->gu_stride / 2, 32, 32))) return rc;
    if ((rc = launch<kMlpGated>(prm, pl, st))) return rc;
    MlpEndParams end{};
    const Result y{a->y, a->y_stride, 0, a->b3, a->residual, a->residual_stride};
    if ((rc = launch_plain(second, y, a->work != nullptr, static_cast<float *>(a->work), &end.of[0], st))) return rc;
    return launch_end(&end, st);
}

size_t kla_b200_mlp_fwd_work_bytes(const kla_b200_mlp_args *a) {
    if (check_sizes(a) || a->rows == 0) return 0;
    return (size_t)partial_words(product_down(*a), device_sms()) * sizeof(float);
}

size_t kla_b200_mlp_work_bytes(const kla_b200_mlp_args *a) {
    if (check_sizes(a) || a->rows == 0) return 0;
    return (size_t)work_of(*a, device_sms()).all * sizeof(float);
}

int kla_b200_mlp_plan(const kla_b200_mlp_args *a, int which, int *columns, int *ctas, int *splits) {
    if (const int rc = check_sizes(a)) return rc;
    if (a->rows == 0 || which < 0 || which > 5 || columns == nullptr || ctas == nullptr || splits == nullptr) return KLA_B200_EINVAL;
    constexpr Product (*products[6])(const kla_b200_mlp_args &) = {product_gate_up, product_down, product_dgu, product_dx, product_dw3, product_dw12};
    const Product p = products[which](*a);
    const Plan pl = plan(p, p.mode != kMlpGated && p.mode != kMlpGrad, device_sms());
    *columns = pl.BN; *ctas = pl.CG; *splits = pl.splits;
    return KLA_B200_OK;
}

int kla_b200_mlp_bwd(const kla_b200_mlp_args *a, void *stream) {
    int rc = check_sizes(a);
    if (rc) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!aligned(a->dw12, 16) || !aligned(a->dw3, 16) || !aligned(a->db12, 2) || !aligned(a->db3, 2) || !aligned(a->work, 16)) return KLA_B200_EALIGN;
    if (a->rows == 0) {
        const struct { void *p; int64_t n; } sums[4] = {{a->dw12, 2 * a->H * a->d}, {a->dw3, a->out * a->H}, {a->db12, 2 * a->H}, {a->db3, a->out}};
        for (const auto &s : sums)
            if (s.p != nullptr) {
                const cudaError_t e = cudaMemsetAsync(s.p, 0, (size_t)s.n * 2, st);
                if (e != cudaSuccess) return entry::cuda_fail(e);
            }
        return KLA_B200_OK;
    }
    const bool inner = a->dx != nullptr || a->dw12 != nullptr || a->db12 != nullptr;
    if ((rc = check_operand(a->dy, a->dy_stride, a->out))) return rc;
    if (inner) {
        if ((rc = check_operand(a->w3, a->w3_stride, a->H)) || (rc = check_operand(a->gu, a->gu_stride, 2 * a->H)) || (rc = check_operand(a->dgu, a->gu_stride, 2 * a->H)))
            return rc;
        if (a->gu_stride % 16) return KLA_B200_EALIGN;
    }
    if (a->dx != nullptr && ((rc = check_operand(a->w12, a->w12_stride, a->d)) || (rc = check_plain(a->dx, a->dx_stride, a->d)))) return rc;
    if (a->dw12 != nullptr && (rc = check_operand(a->x, a->x_stride, a->d))) return rc;
    if (a->dw3 != nullptr && (rc = check_operand(a->h, a->h_stride, a->H))) return rc;
    if ((a->dw12 || a->dw3 || a->db12 || a->db3) && a->work == nullptr) return KLA_B200_EINVAL;
    const int sms = device_sms();
    float *work = static_cast<float *>(a->work);
    const Work at = work_of(*a, sms);
    MlpParams prm;
    MlpEndParams end{};
    MlpSumParams sums{};
    if (a->dw3 != nullptr && (rc = launch_plain(product_dw3(*a), weight(a->dw3, product_dw3(*a)), true, work, &end.of[0], st))) return rc;
    if (inner) {
        const Product dgu = product_dgu(*a);
        const Plan pl = plan(dgu, false, sms);
        if ((rc = fill(&prm, dgu, pl))) return rc;
        prm.act = a->activation;
        prm.side = static_cast<const __nv_bfloat16 *>(a->gu); prm.side_stride = a->gu_stride; prm.side_half = a->gu_stride / 2; prm.side_vec = 1;
        if ((rc = make_map(&prm.map_out, a->dgu, a->H, a->rows, a->gu_stride, 2, a->gu_stride / 2, 32, 32))) return rc;
        if ((rc = launch<kMlpGrad>(prm, pl, st))) return rc;
        if (a->dx != nullptr) {
            const Result dx{a->dx, a->dx_stride, 0, nullptr, nullptr, 0};
            if ((rc = launch_plain(product_dx(*a), dx, work != nullptr, work + at.dx, &end.of[2], st))) return rc;
        }
        if (a->dw12 != nullptr && (rc = launch_plain(product_dw12(*a), weight(a->dw12, product_dw12(*a)), true, work + at.w12, &end.of[1], st))) return rc;
    }
    if (a->db3 != nullptr) sums.of[0] = sum_of(a->dy, a->dy_stride, a->out, 0, 1, work + at.b3, a->db3);
    if (a->db12 != nullptr) sums.of[1] = sum_of(a->dgu, a->gu_stride, a->H, a->gu_stride / 2, 2, work + at.b12, a->db12);
    const int sum_blocks = sums.of[0].blocks + sums.of[1].blocks;
    if (sum_blocks > 0) {
        sums.rows = (int)a->rows;
        sums.stretch_rows = (int)sum_rows(a->rows);
        end.stretches = (int)up(a->rows, sums.stretch_rows);
        if ((rc = launch_behind(kla_mlp_rowsum_kernel, dim3((unsigned)sum_blocks, (unsigned)end.stretches), 256, 0, 1, st, sums))) return rc;
    }
    end.bias[0] = sums.of[0];
    end.bias[1] = sums.of[1];
    return launch_end(&end, st);
}

}  // extern "C"
