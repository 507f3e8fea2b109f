// Entry points of the gated recurrence (kla_gated.cuh): argument checks, kernel and cluster choice, launches.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "../../include/kla_b200.h"
#include "kla_entry.h"
#include "kla_gated.cuh"
#include "kla_launch.cuh"

namespace {

using namespace kla;

bool aligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int check_rows(const kla_b200_tensor3 &t, size_t esz) {
    if (t.ptr == nullptr || t.stride_b < 0 || t.stride_t < 0) return KLA_B200_EINVAL;
    return aligned(t.ptr, esz) ? KLA_B200_OK : KLA_B200_EALIGN;
}
bool pairs(const kla_b200_tensor3 &t, size_t esz) { return aligned(t.ptr, 2 * esz) && t.stride_b % 2 == 0 && t.stride_t % 2 == 0; }
Tensor3 t3(const kla_b200_tensor3 &t) { return Tensor3{t.ptr, t.stride_b, t.stride_t}; }

constexpr int kRanks[] = {1, 2, 3, 4, 5, 6, 8};  // sizes of clusters
constexpr int kRankCount = 7;

// One of the two kernels for a type, alone or in clusters.
struct Kernel {
    void (*kern)(GatedParams);
    int warps, tile;
    size_t smem;  // without the maps of a cluster's CTAs
};
template <typename T, bool PAIR>
Kernel kernel_of(bool backward, bool cluster) {
    using F = GatedFwdShape<T>;
    using B = GatedBwdShape<T>;
    if (backward) return Kernel{cluster ? kla_gated_bwd_kernel<T, PAIR, true> : kla_gated_bwd_kernel<T, PAIR, false>, B::W, kGatedUnit, B::kBytes};
    return Kernel{cluster ? kla_gated_fwd_kernel<T, PAIR, true> : kla_gated_fwd_kernel<T, PAIR, false>, F::W, F::W * F::TS, F::kBytes};
}
Kernel kernel_of(bool bf16, bool pairs, bool backward, bool cluster) {
    if (bf16) return pairs ? kernel_of<__nv_bfloat16, true>(backward, cluster) : kernel_of<__nv_bfloat16, false>(backward, cluster);
    return pairs ? kernel_of<float, true>(backward, cluster) : kernel_of<float, false>(backward, cluster);
}
size_t smem_of(const Kernel &k, int ranks) { return k.smem + (ranks > 1 ? ranks * kGatedCtaMap : 0); }

void fill(cudaLaunchConfig_t *cfg, cudaLaunchAttribute *attr, const Kernel &k, int64_t grid, int ranks, cudaStream_t st) {
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = ranks;
    attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
    *cfg = cudaLaunchConfig_t{};
    cfg->gridDim = dim3((unsigned)grid);
    cfg->blockDim = dim3(k.warps * 32);
    cfg->dynamicSmemBytes = smem_of(k, ranks);
    cfg->stream = st;
    cfg->attrs = attr;
    cfg->numAttrs = ranks > 1 ? 1 : 0;
}

// CTAs that are resident at once by size of cluster; looked up once per device and kernel, which also lets the kernel use its shared
// memory.
struct Slots {
    bool known;
    int ctas[kRankCount];
};
int slots_of(bool bf16, bool pairs, bool backward, Slots *out) {
    static std::mutex mu;
    static Slots table[64][2][2][2];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return entry::cuda_fail(e);
    if (dev < 0 || dev >= 64) return KLA_B200_EUNSUPPORTED;
    std::lock_guard<std::mutex> lock(mu);
    Slots &s = table[dev][bf16][pairs][backward];
    if (!s.known) {
        for (const bool cluster : {false, true}) {
            const Kernel k = kernel_of(bf16, pairs, backward, cluster);
            if ((e = cudaFuncSetAttribute(k.kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_of(k, kGatedMaxCluster))) != cudaSuccess) return entry::cuda_fail(e);
        }
        for (int i = 0; i < kRankCount; ++i) {
            const Kernel k = kernel_of(bf16, pairs, backward, i > 0);
            int n = 0;
            if (i == 0) {
                e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k.kern, k.warps * 32, k.smem);
                n *= device_sms();
            } else {
                cudaLaunchAttribute attr;
                cudaLaunchConfig_t cfg;
                fill(&cfg, &attr, k, 1024 * kRanks[i], kRanks[i], nullptr);
                e = cudaOccupancyMaxActiveClusters(&n, k.kern, &cfg);
                n *= kRanks[i];
            }
            if (e != cudaSuccess) return entry::cuda_fail(e);
            s.ctas[i] = n;
        }
        s.known = true;
    }
    *out = s;
    return KLA_B200_OK;
}

// How many CTAs of a cluster share a sequence: the least time (us) by a model. A round, a tile of each CTA of a cluster, takes `round`
// alone on its SM and by `share` more for the exchange; a second and third CTA on the SM add 35 % each; launching takes `start`; and no
// choice is faster than 80 % of the memory's rate. Of packed sequences the host knows the number and the sum of the lengths (a lone one
// is a batch of one); the longest of n random ones is about ln n + 0.6 times their mean. They take as long as the longest does or as
// all their rounds do with full SMs (half a round of a CTA is left over at each end), and a start per wave. `round` is what makes the
// choice best over 19 shapes, both types and directions, each measured with every size of cluster on B200: 1.7 % slower than the
// best one's kernel on average, 17 % at most. Measured with clusters of 1 / 2 / 4 / 8: forward bfloat16 B=4 L=8192 D=2048 106 / 87 / 103 / 110,
// B=16 L=2048 D=1536 60 / 64 / 71 / 111, B=1 L=8192 D=1024 103 / 67 / 36 / 26, B=8 L=512 D=768 8.7 / 9.1 / 7.9 / 18.3; backward 183 / 155 / 159 / 165,
// 95 / 108 / 115 / 139, 177 / 115 / 61 / 43, 13.8 / 13.6 / 10.6 / 13.4. Packed, clusters of 1 / 2 / 4 / 6 / 8: 40 in 32768 rows of 1536, bfloat16, forward
// 83 / 93 / 113 / 142 / 242, 12 in 32768 of 768 122 / 89 / 65 / 67 / 74, 3 in 65536 of 256 416 / 259 / 138 / 96 / 76, 60 in 2000 of 300, float32, 7 / 13 /
// 19 / 28 / 50, 9 in 6001 of 1024 48 / 36 / 26 / 24 / 36.
int pick_ranks(const Slots &slots, const Kernel &k, int64_t blocks, int64_t rows, int64_t sequences, int64_t L, bool packed, bool backward, size_t esz, int64_t D) {
    packed = packed && sequences > 1;
    const double sms = device_sms();
    const int64_t cells = sequences * blocks;
    const double round = backward ? (esz == 2 ? 1.43 : 2.5) : (esz == 2 ? 1.37 : 1.38);
    constexpr double shares[kRankCount] = {1.0, 1.27, 1.32, 1.37, 1.42, 1.47, 1.6}, starts[kRankCount] = {2.0, 3.5, 4.3, 5.0, 5.3, 5.6, 6.0};
    double steps = (double)L;
    if (packed) steps = std::min(steps, (double)L / sequences * (std::log((double)sequences) + 0.6));
    const double tiles = std::ceil(steps / k.tile), least_us = (double)rows * D * esz * (backward ? 5 : 3) / 5.2e6;
    int best = 1;
    double least = 0.0;
    for (int i = 0; i < kRankCount; ++i) {
        const int r = kRanks[i];
        if (r > 1 && (r > tiles || slots.ctas[i] < r)) continue;
        const double n = (double)cells * r, waves = std::max(1.0, std::ceil(n / slots.ctas[i]));
        const double load = std::min(3.0, std::max(1.0, packed ? n / sms : std::ceil(n / waves / sms))), one = round * shares[i] * (1.0 + 0.35 * (load - 1.0));
        const double own = std::ceil(tiles / r) * one, all = ((double)L * blocks / k.tile + 0.5 * n) * one / (load * sms);
        const double t = packed ? std::max({own, all, least_us}) + waves * starts[i] : std::max(waves * (own + starts[i]), least_us);
        if (r == 1 || t < least) { best = r; least = t; }
    }
    return best;
}

int launch(const Kernel &k, const GatedParams &prm, int64_t sequences, int ranks, cudaStream_t st) {
    const int64_t grid = sequences * prm.blocks * ranks;
    if (grid == 0) return KLA_B200_OK;
    if (grid > 0x7fffffffll) return KLA_B200_EUNSUPPORTED;
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg;
    fill(&cfg, &attr, k, grid, ranks, st);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k.kern, prm);
    if (e != cudaSuccess) return entry::cuda_fail(e);
    entry::count_launch();
    return KLA_B200_OK;
}

// Bytes an asynchronous copy of the tensor's rows may move: 16 where they are aligned so, else 4; 2 of bfloat16 rows that are not in
// pairs.
int width(const kla_b200_tensor3 &t, size_t esz, int64_t D) {
    const int64_t sb = t.stride_b * (int64_t)esz, st = t.stride_t * (int64_t)esz;
    if (aligned(t.ptr, 16) && sb % 16 == 0 && st % 16 == 0) return 16;
    return esz == 4 || (D % 2 == 0 && aligned(t.ptr, 4) && sb % 4 == 0 && st % 4 == 0) ? 4 : 2;
}

int gated(const kla_b200_gated_args *a, void *stream, bool backward) {
    if (a == nullptr || a->B < 0 || a->L < 0 || a->D < 0 || a->sequences < 0) return KLA_B200_EINVAL;
    if (a->dtype != KLA_B200_F32 && a->dtype != KLA_B200_BF16) return KLA_B200_EUNSUPPORTED;
    if (a->B > (1 << 30) || a->L > (1 << 30) || a->D > (1 << 30) || a->sequences > (1 << 30)) return KLA_B200_EUNSUPPORTED;
    const bool packed = a->cu_seqlens != nullptr;
    if (packed ? a->B != 1 : a->sequences != a->B) return KLA_B200_EINVAL;
    const int64_t N = a->sequences;
    if (a->D == 0 || (N == 0 && (!packed || a->L == 0))) return KLA_B200_OK;
    const size_t esz = a->dtype == KLA_B200_BF16 ? 2 : 4;
    const kla_b200_tensor3 *in[5] = {&a->x, &a->gate, backward ? &a->dh : &a->h, &a->dx, &a->dgate};
    bool vec = a->D % 2 == 0;
    if (a->L > 0)
        for (int i = 0; i < (backward ? 5 : 3); ++i) {
            if (const int rc = check_rows(*in[i], esz)) return rc;
            vec = vec && pairs(*in[i], esz);
        }
    if (!backward && N > 0 && a->state_out == nullptr) return KLA_B200_EINVAL;
    if (backward && N > 0 && a->L > 0 && a->ckpt == nullptr) return KLA_B200_EINVAL;
    for (const void *p : {(const void *)a->cu_seqlens, (const void *)a->state, (const void *)a->state_out, (const void *)a->ckpt,
                          (const void *)a->dstate_out, (const void *)a->dstate})
        if (!aligned(p, 4)) return KLA_B200_EALIGN;
    GatedParams prm{};
    prm.N = (int)N; prm.L = (int)a->L; prm.D = (int)a->D;
    prm.blocks = (int)((a->D + kGatedChannels - 1) / kGatedChannels);
    prm.x = t3(a->x); prm.g = t3(a->gate); prm.h = t3(a->h);
    prm.cu = a->cu_seqlens; prm.h0 = a->state; prm.end = a->state_out; prm.ckpt = a->ckpt;
    prm.dh = t3(a->dh); prm.dx = t3(a->dx); prm.dg = t3(a->dgate);
    prm.dend = a->dstate_out; prm.dh0 = a->dstate;
    prm.x_width = width(a->x, esz, a->D); prm.g_width = width(a->gate, esz, a->D); prm.dh_width = width(a->dh, esz, a->D);
    if (const int rc = entry::wait_ctl(&prm.wait)) return rc;
    prm.clears = packed ? (int)std::clamp<int64_t>(a->L / 4096, 1, 16) : 0;
    const int64_t sequences = N + prm.clears;
    Slots slots;
    if (const int rc = slots_of(esz == 2, vec, backward, &slots)) return rc;
    const int ranks = pick_ranks(slots, kernel_of(esz == 2, vec, backward, false), prm.blocks, packed ? a->L : a->B * a->L, N, a->L, packed, backward, esz, a->D);
    return launch(kernel_of(esz == 2, vec, backward, ranks > 1), prm, sequences, ranks, static_cast<cudaStream_t>(stream));
}

}  // namespace

extern "C" {

size_t kla_b200_gated_ckpt_bytes(int64_t sequences, int64_t L, int64_t D, int packed) {
    if (sequences <= 0 || L < 0 || D <= 0) return 0;
    const size_t per = (size_t)((L + kGatedUnit - 1) / kGatedUnit);
    size_t units = packed ? (size_t)(L / kGatedUnit) + (size_t)sequences + 1 : per;
    for (const size_t f : {packed ? (size_t)1 : (size_t)sequences, (size_t)D, sizeof(float)}) {
        if (f != 0 && units > SIZE_MAX / f) return SIZE_MAX;
        units *= f;
    }
    return units;
}

int kla_b200_gated_scan_fwd(const kla_b200_gated_args *args, void *stream) { return gated(args, stream, false); }
int kla_b200_gated_scan_bwd(const kla_b200_gated_args *args, void *stream) { return gated(args, stream, true); }

int kla_b200_gated_step(const kla_b200_gated_step_args *a, void *stream) {
    if (a == nullptr || a->B < 0 || a->D < 0 || a->x_stride_b < 0 || a->gate_stride_b < 0) return KLA_B200_EINVAL;
    if (a->dtype != KLA_B200_F32 && a->dtype != KLA_B200_BF16) return KLA_B200_EUNSUPPORTED;
    if (a->B > (1 << 30) || a->D > (1 << 30)) return KLA_B200_EUNSUPPORTED;
    if (a->B == 0 || a->D == 0) return KLA_B200_OK;
    if (!a->x || !a->gate || !a->state || !a->state_out || !a->h) return KLA_B200_EINVAL;
    const size_t esz = a->dtype == KLA_B200_BF16 ? 2 : 4;
    if (!aligned(a->x, esz) || !aligned(a->gate, esz) || !aligned(a->h, esz) || !aligned(a->state, 4) || !aligned(a->state_out, 4)) return KLA_B200_EALIGN;
    GatedStepParams prm{a->B * a->D, (int)a->D, a->x, a->gate, a->x_stride_b, a->gate_stride_b, a->state, a->state_out, a->h};
    const int64_t grid = (prm.n + 255) / 256;
    if (grid > 0x7fffffffll) return KLA_B200_EUNSUPPORTED;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (esz == 2) kla_gated_step_kernel<__nv_bfloat16><<<(unsigned)grid, 256, 0, st>>>(prm);
    else kla_gated_step_kernel<float><<<(unsigned)grid, 256, 0, st>>>(prm);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return entry::cuda_fail(e);
    entry::count_launch();
    return KLA_B200_OK;
}

}  // extern "C"
