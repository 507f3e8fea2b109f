// The gated feed-forward block on the tensor cores, forward and backward, bfloat16 with float32 accumulation:
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u,  y = h W3^T + b3 (+ residual)
//   dh = dy W3,  dg = dh u act'(g),  du = dh act(g);   dx = [dg du] W12,  dW12 = [dg du]^T x,  dW3 = dy^T h
//
// One kernel takes all six products; what differs is how its operands lie in memory and what its epilogue does:
//   * x Wg^T and x Wu^T are one product whose B tile is rows of Wg beside the same rows of Wu, so that the accumulator holds
//     gate and up of the same columns: the epilogue adds the biases and writes act(g) u (in training g and u, too);
//   * dy W3 turns into dg and du in its epilogue, from the stored g and u;
//   * sums over the rows (the weights' gradients) have few output tiles and a long axis, and so do y and dx of few rows: it is split
//     over CTAs, whose float32 partial sums a second kernel adds in a fixed order (64 rows of 2048 with H = 5456, forward: 35 -> 25 us).
// An operand whose summed axis is not the adjacent one in memory (W3, W12, and both of a weight's gradient) is read as it is, as
// an MN-major operand of the tensor core; nothing is transposed in memory.
//
// A CTA (or a pair of them, which share a tile of 256 rows and each hold half of B's) walks output tiles of 128 x BN. One warp
// issues TMA loads of 64-wide blocks of the summed axis into a ring of blocks, one issues tcgen05.mma from them into one of two
// accumulators in tensor memory, sixteen warps empty the other accumulator meanwhile, through stages of shared memory that TMA
// stores empty. Rows and columns past the ends are zeros of the TMA loads and left out by its stores; widths that are no multiple
// of a tile cost only the padding.
//
// What bounds it: 18 M D H operations forward and backward together for M rows, and for few rows the weights, once from memory. Measured
// at 32768 rows of 768 with H = 2048, forward and backward together: 810 to 840 us a pass in the first twenty of 556 at the rate of a
// library product in a burst of its own (1668 TFLOP/s); 965 to 985 in a loop of a second, at the power limit with the clock at 1.3 to
// 1.4 of 1.97 GHz, of 670 at the rate such products hold there (1384). Each kernel alone, launched one by one: gate and up 126 us
// (1640 TFLOP/s), with gate and up kept 164, down 78, dW3 65, dh and with it dg and du 150, dx 150, dW12 132, the sums' end 11: 750 in all,
// the rest of a pass is the clock's fall. The products
// whose epilogue moves more than an accumulator's worth of data (gate and up kept, dg and du) are bound by that epilogue: at 768
// or 2048 summed elements a tile's products take no longer than its 16 warps take to bring in, work out and send out its data.
#pragma once

#include "kla_common.cuh"

namespace kla {

constexpr int kMlpBM = 128, kMlpBK = 64, kMlpMaxBN = 256;  // rows of a CTA, summed length of a block, columns of a tile
// Sixteen warps empty an accumulator: with eight the latencies of a warp's chunk (of what it fetches, of the accumulator, of its stage,
// of the stores) were not covered, and the gradients of gate and up took 179 us in place of 157 at 32768 rows of 768, H = 2048.
constexpr int kMlpEpiWarps = 16, kMlpThreads = (4 + kMlpEpiWarps) * 32;
constexpr int kMlpStageBytes = 2 * 32 * 64;  // two stages of 32 rows of 64 bytes a warp
constexpr int kMlpRingBytes = 160 * 1024, kMlpMaxStages = 8;
constexpr size_t kMlpSmem = 1024 + kMlpRingBytes + kMlpEpiWarps * kMlpStageBytes + 256;
// A block of the ring: A's rows of a CTA and its share of B's, which in a pair of CTAs is half of them. Rings of 4, 5 and 6 blocks
// of 32 KB measured alike (16384 x 768 x 2048), so that the ring gives way to the sixteen warps' stages.
inline __host__ __device__ int mlp_b_rows(int BN, int cg, bool mn_major) { return mn_major ? (BN / cg + 63) / 64 * 64 : BN / cg; }
inline __host__ __device__ int mlp_block_bytes(int BN, int cg, bool mn_major) { return (kMlpBM + mlp_b_rows(BN, cg, mn_major)) * kMlpBK * 2; }

// wait sites of the status word
constexpr int kMlpSiteEmpty = 0x40, kMlpSiteFull = 0x41, kMlpSiteAccEmpty = 0x42, kMlpSiteAccFull = 0x43, kMlpSiteDrain = 0x44;

enum MlpMode {
    kMlpPlain = 0,   // out = acc (+ bias) (+ residual)
    kMlpGated = 1,   // out = act(gate) up; optionally gate and up themselves
    kMlpGrad = 2,    // out = gradients of gate and up
    kMlpPartial = 3  // float32 sums of a share of the summed axis
};

// How an operand's tile is fetched: rows are the product's m or n.
enum MlpHalves {
    kHalvesNone = 0,
    kHalvesSummed = 1,  // the summed axis is two stretches of `stretch` (third coordinate of the tensor map)
    kHalvesRows = 2,    // the rows are: tiles do not cross
    kHalvesBoth = 3     // a tile is rows of the first beside the same rows of the second (gate and up)
};
struct MlpOperand {
    int mn_major;  // rows are adjacent in memory, not the summed axis
    int halves;
};

struct MlpParams {
    CUtensorMap map_a, map_b;
    CUtensorMap map_out, map_kept;  // gated: h, gate and up; grad: their gradients (map_out). Chunks of 32 columns by 32 rows
    MlpOperand a, b;
    int M, N, K;       // rows, columns (of one half where halves are rows), summed length (of one stretch)
    int BN;            // columns of a tile (gated: of gate and up together)
    int tiles_m, tiles_n, splits;
    int stages;        // blocks of the ring
    int blocks_k;      // 64-wide blocks of the summed axis, all stretches
    int blocks_stretch;
    int act;
    __nv_bfloat16 *out;
    long long out_stride, out_half;  // elements; out_half: to the rows or columns of the second half
    int out_vec;                     // rows can be written 16 bytes at a time
    const __nv_bfloat16 *bias;       // [N], gated [2][N]
    const __nv_bfloat16 *side;       // residual [M, N], grad: gate and up
    long long side_stride, side_half;
    int side_vec;
    int keeps;                       // gated, training: gate and up are kept (map_kept)
    float *partial;                  // [splits][M (both halves)][partial_stride]
    long long partial_stride, partial_rows;
    WaitCtl wait;
};

// A bounded wait without sleeps (mbarrier.try_wait suspends the thread by itself), counted in cycles of at most 2 GHz; gives up like
// mbar_wait. Barriers are addressed by their shared memory address: the ring's two threads run through this once a block, one
// instruction after the other, and are what bounds a block's time as soon as they take more than its products (0.3 us).
__device__ __forceinline__ bool mlp_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mlp_wait(const WaitCtl &w, uint32_t bar, uint32_t parity, int site) {
    if (mlp_try(bar, parity)) return true;
    const long long begin = clock64(), limit = 2ll * w.limit_ns;
    do {
        for (int i = 0; i < 32; ++i)
            if (mlp_try(bar, parity)) return true;
    } while (clock64() - begin < limit);
    atomicCAS(w.status, 0, kStatusWait | site);
    return false;
}
// One lane of a converged warp. The warps that issue loads and products run their loops whole and leave the issuing to this lane by
// a predicate on the instruction: the operands then stay in the uniform registers those instructions take. With a loop of one lane
// every product cost its thread 36 ns of moves between register files and a block's hand-over 155 ns.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r;
}

// Shared memory descriptor of an operand tile in the 128-byte swizzle: 8 rows of 128 bytes make an atom of 1024.
//   summed axis adjacent: a row of 64 summed elements per m or n; atoms of 8 rows follow one another (stride offset)
//   rows adjacent: a line of 64 m or n per summed element; atoms of 8 summed elements follow one another (stride offset), the
//   next 64 rows lie a whole box of 64 x 64 further (leading offset)
__device__ __forceinline__ uint64_t mlp_desc(uint32_t addr, bool mn_major) {
    uint64_t d = (uint64_t)((addr & 0x3ffffu) >> 4);
    d |= (uint64_t)(mn_major ? kMlpBK * 128 / 16 : 1) << 16;
    d |= (uint64_t)(1024 / 16) << 32;
    d |= 1ull << 46;  // sm_100
    d |= 2ull << 61;  // 128-byte swizzle
    return d;
}

template <int CG>
__device__ __forceinline__ void mlp_mma(uint32_t on, uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n.reg .pred p, q;\nsetp.ne.u32 p, %4, 0;\nsetp.ne.u32 q, %5, 0;\n"
            "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(acc), "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(on)
            : "memory");
    else
        asm volatile(
            "{\n.reg .pred p, q;\nsetp.ne.u32 p, %4, 0;\nsetp.ne.u32 q, %5, 0;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(acc), "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(on)
            : "memory");
}
// an arrival at the barrier, in a pair at both CTAs', when the products issued so far are done
template <int CG>
__device__ __forceinline__ void mlp_commit(uint32_t on, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\n"
            "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n" ::"r"(bar), "h"((uint16_t)3), "r"(on)
            : "memory");
    else
        asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %1, 0;\n@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar), "r"(on) : "memory");
}
// the address that `addr` has in the pair's first CTA
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
// Without release semantics, which would wait for the warp's stores to memory: what the arrival reports, that the accumulator has
// been read, is complete (tcgen05.wait::ld) and fenced before it.
template <int CG>
__device__ __forceinline__ void mlp_arrive_leader(uint32_t bar) {
    if constexpr (CG == 2) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_leader(bar)) : "memory");
    else asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mlp_expect(uint32_t on, uint32_t bar, uint32_t bytes) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\n@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}\n" ::"r"(bar), "r"(bytes), "r"(on) : "memory");
}
template <int CG>
__device__ __forceinline__ void mlp_load(uint32_t on, uint32_t dst, uint64_t tm, int x, int y, int z, uint32_t bar) {  // bar: the leader's
    if constexpr (CG == 2)
        asm volatile(
            "{\n.reg .pred q;\nsetp.ne.u32 q, %6, 0;\n"
            "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%2, %3, %4}], [%5];\n}\n" ::"r"(dst), "l"(tm), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(on)
            : "memory");
    else
        asm volatile(
            "{\n.reg .pred q;\nsetp.ne.u32 q, %6, 0;\n"
            "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%2, %3, %4}], [%5];\n}\n" ::"r"(dst), "l"(tm), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(on)
            : "memory");
}
// A warp's stage (32 rows of 32 columns, 64-byte swizzle) to memory by one lane's copy, which clips what lies outside; all lanes have
// written their rows. The stage may be written again after mlp_stored.
__device__ __forceinline__ void mlp_store(const CUtensorMap *tm, const void *stage, int x, int y, int z, int lane) {
    if (lane == 0)
        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(z),
                     "r"(smem_u32(stage))
                     : "memory");
}
__device__ __forceinline__ void mlp_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void mlp_stored() {  // (lanes that issued nothing pass)
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}
__device__ __forceinline__ void mlp_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_load8(float2 (&v)[4], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0].x), "=f"(v[0].y), "=f"(v[1].x), "=f"(v[1].y), "=f"(v[2].x), "=f"(v[2].y), "=f"(v[3].x), "=f"(v[3].y)
                 : "r"(addr));
}
// The loads have arrived; the registers pass through, so that nothing is taken from them before.
__device__ __forceinline__ void tmem_load_wait(float2 (&v)[4]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+f"(v[0].x), "+f"(v[0].y), "+f"(v[1].x), "+f"(v[1].y), "+f"(v[2].x), "+f"(v[2].y), "+f"(v[3].x), "+f"(v[3].y)::"memory");
}
// behind a wait already made
__device__ __forceinline__ void tmem_loaded(float2 (&v)[4]) {
    asm volatile("" : "+f"(v[0].x), "+f"(v[0].y), "+f"(v[1].x), "+f"(v[1].y), "+f"(v[2].x), "+f"(v[2].y), "+f"(v[3].x), "+f"(v[3].y)::"memory");
}
__device__ __forceinline__ void tcgen05_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A warp's stage: 32 rows of 64 bytes. Rows go in and out a row per lane; memory is walked four lanes to a row. The 16-byte pieces
// of a row change places with the row's number, which keeps both ways free of bank conflicts. The caller puts __syncwarp() between
// the two.
struct MlpStage {
    char *base;
    int lane;
    __device__ __forceinline__ char *piece(int row, int i) const { return base + row * 64 + (i ^ (row >> 1 & 3)) * 16; }
    __device__ __forceinline__ void put_row(const uint4 (&v)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4 *>(piece(lane, i)) = v[i];
    }
    // E: element type; rows x cols of them are there
    template <typename E>
    __device__ __forceinline__ void store(E *p, long long stride, int rows, int cols, bool vec) const {
        constexpr int per = 16 / sizeof(E);
        const int r0 = lane / 4, c = lane % 4 * per;
        const char *from = piece(r0, lane % 4);  // rows 8 apart hold a piece at the same place
        E *to = p + r0 * stride + c;
        if (vec && cols >= 4 * per) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4 *>(from + i * 8 * 64);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r0 + 8 * i < rows) *reinterpret_cast<uint4 *>(to + i * 8 * stride) = v[i];
        } else {
            for (int i = 0; i < 4; ++i)
                if (r0 + 8 * i < rows) {
#pragma unroll
                    for (int e = 0; e < per; ++e)
                        if (c + e < cols) to[i * 8 * stride + e] = reinterpret_cast<const E *>(from + i * 8 * 64)[e];
                }
        }
    }
    // what store would write, from memory into registers; zeros where there is nothing
    __device__ __forceinline__ void fetch(uint4 (&v)[4], const __nv_bfloat16 *p, long long stride, int rows, int cols, bool vec) const {
        const int r0 = lane / 4, c = lane % 4 * 8;
        const __nv_bfloat16 *from = p + r0 * stride + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (vec && cols >= 32) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r0 + 8 * i < rows) v[i] = __ldg(reinterpret_cast<const uint4 *>(from + i * 8 * stride));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r0 + 8 * i < rows) {
                    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (c + e < cols) w[e / 2] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short *>(from + i * 8 * stride) + e) << (e % 2 * 16);
                    v[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
        }
    }
    __device__ __forceinline__ void put_fetched(const uint4 (&v)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4 *>(piece(i * 8 + lane / 4, lane % 4)) = v[i];
    }
};
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Gate and up as the backward finds them: 16 bits with a sign, six of exponent and nine of mantissa. Rounded to bfloat16 their
// two roundings would be half of the error of a gradient (0.0030 of dx and dW12 in the 2-norm, against 0.0017 of rounding
// the result alone); nine bits leave the rounding of the gradients that go into the products (0.0025). 2^-31 to 2^32 at full
// accuracy, steps of 2^-40 below; what is larger, infinite or NaN comes back as NaN. (A value times 2^-95 has its 2^-31 at the least
// normal number, 2^-126, and 14 bits dropped of 2^-149 below are steps of 2^-135.)
constexpr uint32_t kKeptTop = 0x7fffu << 14;
// the code in the upper half, s being x 2^-95; the least of its size and kKeptTop makes NaN the top code, too
__device__ __forceinline__ uint32_t keep(float x, float s) {
    const float m = fminf(fabsf(s), __uint_as_float(kKeptTop));
    return __float_as_uint(m) * 4u + 0x8000u | __float_as_uint(x) & 0x80000000u;
}
__device__ __forceinline__ uint32_t keep2(float2 x) {
    const float2 s = mul2(x, dup2(0x1p-95f));
    return __byte_perm(keep(x.x, s.x), keep(x.y, s.y), 0x7632);
}
__device__ __forceinline__ float2 kept2(uint32_t w) {
    const uint32_t lo = (uint32_t)((int32_t)(w << 16) >> 2) & 0x9fffc000u, hi = (uint32_t)((int32_t)w >> 2) & 0x9fffc000u;
    const float2 v = mul2(make_float2(__uint_as_float(lo), __uint_as_float(hi)), dup2(0x1p95f));
    const float nan = __uint_as_float(0x7fffffffu);
    return make_float2((lo & 0x7fffffffu) == kKeptTop ? nan : v.x, (hi & 0x7fffffffu) == kKeptTop ? nan : v.y);
}

__device__ __forceinline__ float mlp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The activation and its derivative. Which one is chosen once for 32 columns, not per element: with the choice (and gelu's error
// function) inside the unrolled loops their code left the instruction cache, and the gated product took 288 us in place of 193, the
// one of the gradients 342 in place of 197 (32768 rows of 768, H = 2048).
template <int ACT, bool SLOPE>
__device__ __forceinline__ void mlp_act(float g, float &f, float &df) {
    if (ACT == 1) {  // gelu
        const float cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        f = g * cdf;
        if (SLOPE) df = fmaf(g * 0.3989422804014327f, mlp_ex2(-0.72134752044448170f * g * g), cdf);
    } else if (ACT == 2) {  // relu; NaN stays
        f = g < 0.0f ? 0.0f : g;
        if (SLOPE) df = g > 0.0f ? 1.0f : 0.0f;
    } else {
        f = g;
        if (SLOPE) df = 1.0f;
    }
}
template <int ACT, bool SLOPE>
__device__ __forceinline__ void mlp_act2(float2 g, float2 &f, float2 &df) {
    if (ACT == 0) {  // silu, in paired instructions: what bounds these epilogues is instruction issue
        const float2 e = mul2(g, dup2(-1.4426950408889634f)), d = add2(make_float2(mlp_ex2(e.x), mlp_ex2(e.y)), dup2(1.0f));
        const float2 s = make_float2(rcp_approx(d.x), rcp_approx(d.y));
        f = mul2(g, s);
        if (SLOPE) df = fma2(f, fma2(s, dup2(-1.0f), dup2(1.0f)), s);
    } else {
        mlp_act<ACT, SLOPE>(g.x, f.x, df.x);
        mlp_act<ACT, SLOPE>(g.y, f.y, df.y);
    }
}
// A gate as it is kept: where the activation closes (silu, gelu and relu of large negative gates) its size says nothing, the value and the
// slope are 0 whatever it is. It is kept as a gate that closes and has a code, so that a hidden unit masked by a bias of the
// type's lowest value gets its gradients of 0. NaN and what is NaN forward (silu and gelu of -inf) stay NaN.
constexpr float kClosedGate = -0x1p20f;
template <int ACT>
__device__ __forceinline__ float2 gate_to_keep(float2 g) {
    if (ACT == 2) {
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(g.x) : "f"(kClosedGate));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(g.y) : "f"(kClosedGate));
        return g;
    }
    if (ACT == 3) return g;
    return fma2(g, dup2(0.0f), make_float2(fmaxf(g.x, kClosedGate), fmaxf(g.y, kClosedGate)));
}
template <int ACT>
__device__ __forceinline__ uint4 keep8_gates(const float2 (&g)[4]) {
    return make_uint4(keep2(gate_to_keep<ACT>(g[0])), keep2(gate_to_keep<ACT>(g[1])), keep2(gate_to_keep<ACT>(g[2])), keep2(gate_to_keep<ACT>(g[3])));
}
__device__ __forceinline__ uint4 pack8(const float2 (&x)[4]) { return make_uint4(pack2(x[0].x, x[0].y), pack2(x[1].x, x[1].y), pack2(x[2].x, x[2].y), pack2(x[3].x, x[3].y)); }
__device__ __forceinline__ uint4 keep8(const float2 (&x)[4]) { return make_uint4(keep2(x[0]), keep2(x[1]), keep2(x[2]), keep2(x[3])); }
// cols: of the eight that exist
__device__ __forceinline__ void add_bias(float2 (&x)[4], const __nv_bfloat16 *bias, int cols) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (2 * j < cols) x[j].x += __bfloat162float(bias[2 * j]);
        if (2 * j + 1 < cols) x[j].y += __bfloat162float(bias[2 * j + 1]);
    }
}
// A chunk of 32 columns of a row: f is called for its four pieces of eight columns, the accumulator's (and, TWO, those of a second
// place in it) on their way a piece ahead.
template <bool TWO, typename F>
__device__ __forceinline__ void mlp_pieces(uint32_t acc, uint32_t acc2, F &&f) {
    float2 a[4], b[4], x[4], y[4];
    tmem_load8(a, acc);
    if (TWO) tmem_load8(b, acc2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        tmem_load_wait(a);
        if (TWO) tmem_loaded(b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = a[j];
            if (TWO) y[j] = b[j];
        }
        if (i < 3) {
            tmem_load8(a, acc + 8 * (i + 1));
            if (TWO) tmem_load8(b, acc2 + 8 * (i + 1));
        }
        f(i, x, y);
    }
}
// act(gate) up of a chunk to h; gate and up to the warp's stages where they are kept.
template <int ACT>
__device__ __forceinline__ void mlp_gated_chunk(uint32_t gate, uint32_t up, const __nv_bfloat16 *bias, int N, int cols, bool kept, const MlpStage &st, const MlpStage &st2,
                                                uint4 (&h)[4]) {
    mlp_pieces<true>(gate, up, [&](int i, float2 (&g)[4], float2 (&u)[4]) {
        if (bias != nullptr) {
            add_bias(g, bias + 8 * i, cols - 8 * i);
            add_bias(u, bias + N + 8 * i, cols - 8 * i);
        }
        if (kept) {
            *reinterpret_cast<uint4 *>(st.piece(st.lane, i)) = keep8_gates<ACT>(g);
            *reinterpret_cast<uint4 *>(st2.piece(st.lane, i)) = keep8(u);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 f, df;
            mlp_act2<ACT, false>(g[j], f, df);
            g[j] = mul2(f, u[j]);
        }
        h[i] = pack8(g);
    });
}
// The gradients of gate and up of a row's eight columns, in place of the kept gate and up.
template <int ACT>
__device__ __forceinline__ void mlp_slopes(const float2 (&dh)[4], uint4 &gate, uint4 &up) {
    uint32_t *g = reinterpret_cast<uint32_t *>(&gate), *u = reinterpret_cast<uint32_t *>(&up);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float2 f, df;
        mlp_act2<ACT, true>(kept2(g[j]), f, df);
        const float2 dg = mul2(mul2(dh[j], kept2(u[j])), df), du = mul2(dh[j], f);
        g[j] = pack2(dg.x, dg.y);
        u[j] = pack2(du.x, du.y);
    }
}
// ... of a chunk: dh from the accumulator, the kept ones from the warp's two stages.
template <int ACT>
__device__ __forceinline__ void mlp_slopes_chunk(uint32_t acc, const MlpStage &st, const MlpStage &st2) {
    float2 next[4];
    tmem_load8(next, acc);
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        float2 dh[4];
        tmem_load_wait(next);
#pragma unroll
        for (int j = 0; j < 4; ++j) dh[j] = next[j];
        if (i < 3) tmem_load8(next, acc + 8 * (i + 1));
        uint4 *pg = reinterpret_cast<uint4 *>(st.piece(st.lane, i)), *pu = reinterpret_cast<uint4 *>(st2.piece(st.lane, i));
        uint4 g = *pg, u = *pu;
        mlp_slopes<ACT>(dh, g, u);
        *pg = g;
        *pu = u;
    }
}

constexpr int kMlpGroup = 8;
struct MlpTile {
    int m, n, split;    // first row (of its half), first column (gated: of gate), share of the summed axis
    int m_half;
    int k0, k1;         // blocks
};
template <int CG>
__device__ __forceinline__ MlpTile mlp_tile(const MlpParams &p, int t) {
    MlpTile r;
    const int per = p.tiles_m * p.tiles_n;
    r.split = t / per;
    t -= r.split * per;
    // tiles side by side in time are a block of tiles, so that their operands meet in L2: kMlpGroup rows of tiles, column after column
    const int first = t / (kMlpGroup * p.tiles_n) * kMlpGroup, high = min(kMlpGroup, p.tiles_m - first);
    t -= first * p.tiles_n;
    const int tn = t / high, tm = first + t - tn * high;
    const int per_half = p.a.halves == kHalvesRows ? p.tiles_m / 2 : p.tiles_m;
    r.m_half = tm / per_half;
    r.m = (tm - r.m_half * per_half) * kMlpBM * CG;
    r.n = tn * (p.b.halves == kHalvesBoth ? p.BN / 2 : p.BN);
    r.k0 = (int)((long long)p.blocks_k * r.split / p.splits);
    r.k1 = (int)((long long)p.blocks_k * (r.split + 1) / p.splits);
    return r;
}

template <int MODE, int CG>
__global__ void __launch_bounds__(kMlpThreads, 1) kla_mlp_kernel(const __grid_constant__ MlpParams prm) {
    extern __shared__ char raw[];
    char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    constexpr int W = kMlpEpiWarps, PARTS = W / 4;
    char *epi = smem + kMlpRingBytes;
    const int S = prm.stages, block_bytes = mlp_block_bytes(prm.BN, CG, prm.b.mn_major);
    // full, acc_empty: of the leader (the pair's first CTA); empty, acc_full: of each CTA
    uint64_t *full = reinterpret_cast<uint64_t *>(epi + W * kMlpStageBytes), *empty = full + kMlpMaxStages, *acc_full = empty + kMlpMaxStages, *acc_empty = acc_full + 2, *drain = acc_empty + 2;
    uint32_t *tmem_at = reinterpret_cast<uint32_t *>(drain + 1);
    int *failed = reinterpret_cast<int *>(tmem_at + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;  // (known to be uniform)
    uint32_t rank = 0;
    if (CG == 2) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int first = blockIdx.x / CG, step = gridDim.x / CG;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], W * CG); }
        mbar_init(drain, 1);
        *failed = 0;
        mbar_fence_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&prm.map_a)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&prm.map_b)) : "memory");
    }
    if (warp == 2) {
        if constexpr (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tcgen05_before_sync();
    if constexpr (CG == 2) mlp_cluster_sync();
    else __syncthreads();
    tcgen05_after_sync();
    const uint32_t tmem = *tmem_at;
    // what stands above runs beside the end of the kernel in front (programmatic dependent launch); memory is touched from here on
    grid_dep_launch();
    grid_dep_wait();
    const int tiles = prm.tiles_m * prm.tiles_n * prm.splits;
    int issued = 0;  // producer: blocks whose loads were issued

    const uint32_t smem_at = smem_u32(smem), full_at = smem_u32(full), empty_at = smem_u32(empty), acc_full_at = smem_u32(acc_full), acc_empty_at = smem_u32(acc_empty);

    if (warp == 0) {
        const uint32_t on = elect_one();
        const WaitCtl wait = prm.wait;
        const uint64_t map_a = reinterpret_cast<uint64_t>(&prm.map_a), map_b = reinterpret_cast<uint64_t>(&prm.map_b);
        const bool a_lines = prm.a.mn_major != 0, b_lines = prm.b.mn_major != 0;
        // B's rows of this CTA; a gated pair's first CTA has gate's, its second up's, a CTA alone both, one behind the other
        const bool both = prm.b.halves == kHalvesBoth, a_rows_half = prm.a.halves == kHalvesRows;
        const int b_rows = prm.BN / CG / (both && CG == 1 ? 2 : 1), b_first = both ? 0 : (int)rank * b_rows, stretch_blocks = prm.blocks_stretch;
        const uint32_t bytes = CG * block_bytes, leader_full = CG == 2 ? in_leader(full_at) : full_at;
        int s = 0;
        uint32_t phase = 1;  // the ring begins empty: a wait for the phase before the first passes
        bool ok = true;
        for (int t = first; ok && t < tiles; t += step) {
            const MlpTile tl = mlp_tile<CG>(prm, t);
            int stretch = tl.k0 / stretch_blocks, kb = tl.k0 - stretch * stretch_blocks;
            const int m = tl.m + (int)rank * kMlpBM, n = tl.n + b_first;
            for (int left = tl.k1 - tl.k0; left > 0; --left) {
                if (!mlp_wait(wait, empty_at + 8 * s, phase, kMlpSiteEmpty) || issued == wait.skip_tile) {  // skip_tile: the tests'
                    ok = false;                                                                            // incomplete hand-over
                    break;
                }
                const uint32_t at_a = smem_at + s * block_bytes, at_b = at_a + kMlpBM * kMlpBK * 2, bar = leader_full + 8 * s;
                const int k = kb * kMlpBK, za = a_rows_half ? tl.m_half : stretch, zb = both ? (int)rank : stretch;
                if (rank == 0) mlp_expect(on, full_at + 8 * s, bytes);
                if (a_lines) {
                    mlp_load<CG>(on, at_a, map_a, m, k, za, bar);
                    mlp_load<CG>(on, at_a + 64 * 128, map_a, m + 64, k, za, bar);
                } else {
                    mlp_load<CG>(on, at_a, map_a, k, m, za, bar);
                }
                if (b_lines) {
                    for (int r = 0; r < b_rows; r += 64) mlp_load<CG>(on, at_b + r * 128, map_b, n + r, k, zb, bar);
                } else {
                    mlp_load<CG>(on, at_b, map_b, k, n, zb, bar);
                    if (both && CG == 1) mlp_load<CG>(on, at_b + b_rows * 128, map_b, k, n, 1, bar);
                }
                ++issued;
                if (++s == S) { s = 0; phase ^= 1; }
                if (++kb == stretch_blocks) { kb = 0; ++stretch; }
            }
        }
        if (!ok && lane == 0) *failed = 1;
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t on = elect_one();
            const WaitCtl wait = prm.wait;
            // float32 accumulators of bfloat16 operands; majors; N / 8; M / 16
            const uint32_t idesc = 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(prm.a.mn_major != 0) << 15 | (uint32_t)(prm.b.mn_major != 0) << 16 |
                                   (uint32_t)(prm.BN / 8) << 17 | (uint32_t)(kMlpBM * CG / 16) << 24;
            const uint32_t step_a = (prm.a.mn_major ? 2048 : 32) / 16, step_b = (prm.b.mn_major ? 2048 : 32) / 16;
            const uint64_t desc_a = mlp_desc(smem_at, prm.a.mn_major), desc_b = mlp_desc(smem_at + kMlpBM * kMlpBK * 2, prm.b.mn_major);
            int s = 0;
            uint32_t phase = 0, acc = 0, acc_phase = 1;
            bool ok = true;
            for (int t = first; ok && t < tiles; t += step) {
                const MlpTile tl = mlp_tile<CG>(prm, t);
                if (!mlp_wait(wait, acc_empty_at + 8 * acc, acc_phase, kMlpSiteAccEmpty)) { ok = false; break; }
                tcgen05_after_sync();
                const uint32_t d = tmem + acc * kMlpMaxBN;
                uint32_t add = 0;
                for (int left = tl.k1 - tl.k0; left > 0; --left) {
                    if (!mlp_wait(wait, full_at + 8 * s, phase, kMlpSiteFull)) { ok = false; break; }
                    tcgen05_after_sync();
                    const uint64_t da = desc_a + (uint32_t)(s * block_bytes / 16), db = desc_b + (uint32_t)(s * block_bytes / 16);
#pragma unroll
                    for (int i = 0; i < kMlpBK / 16; ++i) {
                        mlp_mma<CG>(on, d, da + i * step_a, db + i * step_b, idesc, add);
                        add = 1;
                    }
                    mlp_commit<CG>(on, empty_at + 8 * s);
                    if (++s == S) { s = 0; phase ^= 1; }
                }
                if (ok) mlp_commit<CG>(on, acc_full_at + 8 * acc);
                if (++acc == 2) { acc = 0; acc_phase ^= 1; }
            }
            if (!ok && lane == 0) *failed = 1;
        }
    } else if (warp >= 4) {
        const int quad = warp % 4, part = (warp - 4) / 4;
        const MlpStage st{epi + (warp - 4) * kMlpStageBytes, lane}, st2{st.base + 32 * 64, lane};
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        // chunks of 32 columns are dealt to the warps of a quarter of the rows in turn
        const int width = MODE == kMlpGated ? prm.BN / 2 : prm.BN, c0 = part * 32, cstep = PARTS * 32;
        const int row0 = (int)rank * kMlpBM + quad * 32;
        // what the epilogue reads besides the accumulator is fetched a chunk of 32 columns ahead, the next tile's first during the
        // wait for its accumulator
        uint4 f1[4], f2[4];
        auto fetch = [&](int m, int n) {
            if (MODE == kMlpPlain && prm.side != nullptr) st.fetch(f1, prm.side + (long long)m * prm.side_stride + n, prm.side_stride, prm.M - m, prm.N - n, prm.side_vec);
            if (MODE == kMlpGrad) {
                const __nv_bfloat16 *p = prm.side + (long long)m * prm.side_stride + n;
                st.fetch(f1, p, prm.side_stride, prm.M - m, prm.N - n, true);
                st.fetch(f2, p + prm.side_half, prm.side_stride, prm.M - m, prm.N - n, true);
            }
        };
        uint32_t acc = 0, acc_phase = 0;
        for (int t = first; t < tiles; t += step) {
            const MlpTile tl = mlp_tile<CG>(prm, t);
            const int m = tl.m + row0, rows = prm.M - m;
            if (c0 < width) fetch(m, tl.n + c0);
            if (MODE == kMlpGrad && t + step < tiles) {  // the next tile's gate and up into L2: a chunk ahead covers L2's latency only
                const MlpTile nx = mlp_tile<CG>(prm, t + step);
                const int nm = nx.m + row0 + lane, nn = nx.n + c0;
                if (nm < prm.M) {
                    const __nv_bfloat16 *p = prm.side + (long long)nm * prm.side_stride + nn;
                    for (int c = 0; c0 + c < width && nn + c < prm.N; c += cstep) {
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(p + c));
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(p + prm.side_half + c));
                    }
                }
            }
            bool ok = true;
            if (lane == 0) ok = mlp_wait(prm.wait, acc_full_at + 8 * acc, acc_phase, kMlpSiteAccFull);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) {
                if (lane == 0) *failed = 1;
                break;
            }
            tcgen05_after_sync();
            const uint32_t d = tmem + acc * kMlpMaxBN + lanes, acc_done = acc_empty_at + 8 * acc;
            if (++acc == 2) { acc = 0; acc_phase ^= 1; }
            if (c0 >= width) {
                __syncwarp();
                if (lane == 0) mlp_arrive_leader<CG>(acc_done);
            }
            for (int c = c0; c < width; c += cstep) {
                const int n = tl.n + c, cols = prm.N - n;
                auto done = [&] {  // behind the last read of the accumulator
                    if (c + cstep >= width) {
                        tcgen05_before_sync();
                        __syncwarp();
                        if (lane == 0) mlp_arrive_leader<CG>(acc_done);
                    }
                };
                __nv_bfloat16 *out = prm.out + tl.m_half * prm.out_half + (long long)m * prm.out_stride + n;
                if constexpr (MODE == kMlpGrad) {
                    mlp_stored();  // of the chunk before
                    st.put_fetched(f1);
                    st2.put_fetched(f2);
                    __syncwarp();
                    if (c + cstep < width) fetch(m, n + cstep);
                    if (prm.act == 0) mlp_slopes_chunk<0>(d + c, st, st2);
                    else if (prm.act == 1) mlp_slopes_chunk<1>(d + c, st, st2);
                    else if (prm.act == 2) mlp_slopes_chunk<2>(d + c, st, st2);
                    else mlp_slopes_chunk<3>(d + c, st, st2);
                    done();
                    fence_proxy_async();
                    __syncwarp();
                    if (cols > 0 && rows > 0) {
                        mlp_store(&prm.map_out, st.base, n, m, 0, lane);
                        mlp_store(&prm.map_out, st2.base, n, m, 1, lane);
                    }
                    mlp_store_commit();
                    continue;
                }
                const __nv_bfloat16 *bias = prm.bias != nullptr ? prm.bias + n : nullptr;
                if constexpr (MODE == kMlpGated) {
                    uint4 h[4];
                    const bool keeps = prm.keeps != 0;
                    mlp_stored();
                    if (prm.act == 0) mlp_gated_chunk<0>(d + c, d + width + c, bias, prm.N, cols, keeps, st, st2, h);
                    else if (prm.act == 1) mlp_gated_chunk<1>(d + c, d + width + c, bias, prm.N, cols, keeps, st, st2, h);
                    else if (prm.act == 2) mlp_gated_chunk<2>(d + c, d + width + c, bias, prm.N, cols, keeps, st, st2, h);
                    else mlp_gated_chunk<3>(d + c, d + width + c, bias, prm.N, cols, keeps, st, st2, h);
                    done();
                    const bool some = rows > 0;
                    if (keeps) {
                        fence_proxy_async();
                        __syncwarp();
                        if (some) {
                            mlp_store(&prm.map_kept, st.base, n, m, 0, lane);
                            mlp_store(&prm.map_kept, st2.base, n, m, 1, lane);
                        }
                        mlp_store_commit();
                        mlp_stored();
                    }
                    st.put_row(h);
                    fence_proxy_async();
                    __syncwarp();
                    if (some) mlp_store(&prm.map_out, st.base, n, m, 0, lane);
                    mlp_store_commit();
                    continue;
                } else if constexpr (MODE == kMlpPartial) {
                    // four of a row's 16-byte pieces in either stage
                    mlp_pieces<false>(d + c, 0u, [&](int i, float2 (&x)[4], float2 (&)[4]) {
                        const MlpStage &to = i < 2 ? st : st2;
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            *reinterpret_cast<float4 *>(to.piece(lane, i % 2 * 2 + e)) = make_float4(x[2 * e].x, x[2 * e].y, x[2 * e + 1].x, x[2 * e + 1].y);
                    });
                    done();
                    __syncwarp();
                    float *p = prm.partial + (long long)tl.split * prm.partial_rows * prm.partial_stride +
                               ((long long)tl.m_half * prm.M + m) * prm.partial_stride + n;
                    st.store(p, prm.partial_stride, rows, cols, true);
                    st2.store(p + 16, prm.partial_stride, rows, cols - 16, true);
                } else {
                    const bool side = prm.side != nullptr;
                    if (side) {
                        st.put_fetched(f1);
                        __syncwarp();
                        if (c + cstep < width) fetch(m, n + cstep);
                    }
                    mlp_pieces<false>(d + c, 0u, [&](int i, float2 (&x)[4], float2 (&)[4]) {
                        uint4 *p = reinterpret_cast<uint4 *>(st.piece(lane, i));
                        if (bias != nullptr) add_bias(x, bias + 8 * i, cols - 8 * i);
                        if (side) {
                            const uint4 r = *p;
                            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) x[j] = add2(x[j], make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u)));
                        }
                        *p = pack8(x);
                    });
                    done();
                    __syncwarp();
                    st.store(out, prm.out_stride, rows, cols, prm.out_vec);
                }
                __syncwarp();
            }
        }
    }
    if (MODE == kMlpGated || MODE == kMlpGrad) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // own stores are done
    __syncwarp();
    if constexpr (CG == 2) mlp_cluster_sync();
    else __syncthreads();
    int bad = *failed;
    if constexpr (CG == 2) {
        uint32_t there;
        int other;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_u32(failed)), "r"(rank ^ 1u));
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(other) : "r"(there) : "memory");
        bad |= other;
    }
    if (bad) {  // a wait ran out: copies and products still under way end, or get as long again, before their memory is given back
        if (warp == 0 && lane == 0 && rank == 0)
            for (int b = max(0, issued - S); b < issued; ++b) mlp_wait(prm.wait, full_at + 8 * (b % S), (b / S) & 1, kMlpSiteDrain);
        if (warp == 1 && rank == 0) {
            mlp_commit<CG>(elect_one(), smem_u32(drain));
            mlp_wait(prm.wait, smem_u32(drain), 0, kMlpSiteDrain);
        }
        __syncwarp();
    }
    tcgen05_before_sync();
    if constexpr (CG == 2) mlp_cluster_sync();
    else __syncthreads();
    if (warp == 2) {
        tcgen05_after_sync();
        if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// Sums over rows of bfloat16 matrices (the biases' gradients) whose rows are 16-byte aligned: a block adds 256 columns of a stretch of
// rows, eight rows side by side and eight columns a thread by one access, into float32 [stretches][total]. `blocks` blocks of columns
// are of the first matrix, the others of the second (gate's and up's gradients are one matrix of two halves half_gap apart).
constexpr int kMlpSumCols = 256;
struct MlpSum {
    const __nv_bfloat16 *x;
    long long stride, half_gap;
    int cols, half_blocks, blocks, total;  // cols, half_blocks: of one half; blocks, total: of all
    float *partial;
    __nv_bfloat16 *out;
};
struct MlpSumParams {
    MlpSum of[2];
    int rows, stretch_rows;
};
__global__ void __launch_bounds__(256) kla_mlp_rowsum_kernel(const __grid_constant__ MlpSumParams prm) {
    __shared__ float part[8][kMlpSumCols];
    grid_dep_launch();
    grid_dep_wait();
    const bool second = (int)blockIdx.x >= prm.of[0].blocks;
    const MlpSum &m = prm.of[second];
    const int bx = blockIdx.x - (second ? prm.of[0].blocks : 0), half = bx / m.half_blocks, c0 = (bx - half * m.half_blocks) * kMlpSumCols;
    const int g = threadIdx.x / 32, c = c0 + threadIdx.x % 32 * 8;
    const int r0 = blockIdx.y * prm.stretch_rows + g, r1 = min(prm.rows, ((int)blockIdx.y + 1) * prm.stretch_rows);
    const __nv_bfloat16 *x = m.x + half * m.half_gap + c;
    float s[8] = {};
    if (c + 8 <= m.cols) {
#pragma unroll 8
        for (int r = r0; r < r1; r += 8) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(x + r * m.stride));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[2 * e] += __uint_as_float(w[e] << 16);
                s[2 * e + 1] += __uint_as_float(w[e] & 0xffff0000u);
            }
        }
    } else {
        for (int r = r0; r < r1; r += 8)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < m.cols) s[e] += __bfloat162float(x[r * m.stride + e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) part[g][threadIdx.x % 32 * 8 + e] = s[e];
    __syncthreads();
    const int col = c0 + threadIdx.x;
    if (col < m.cols) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += part[i][threadIdx.x];
        m.partial[(long long)blockIdx.y * m.total + half * m.cols + col] = t;
    }
}

// The end of split products, one launch for all of a backward: the partial sums of up to three products, four columns a thread, and those
// of the biases' gradients, 32 columns a block and every eighth stretch a warp; each in a fixed order. A product's bias and residual
// are added here in float32, in the order of the unsplit product's epilogue.
struct MlpReduce {
    const float *partial;
    long long split_stride, stride;  // elements; stride a multiple of 4
    int splits, rows, cols, blocks;  // blocks: of the grid, up to this one's last
    __nv_bfloat16 *out;
    long long out_stride;
    int vec;                         // four columns of a row of `out` can be written at once
    const __nv_bfloat16 *bias, *side;  // or nullptr
    long long side_stride;
};
constexpr int kMlpSums = 3;
struct MlpEndParams {
    MlpReduce of[kMlpSums];
    MlpSum bias[2];
    int bias_blocks, stretches;      // bias_blocks: of the grid, up to the first bias's last
};
__global__ void __launch_bounds__(256) kla_mlp_end_kernel(const __grid_constant__ MlpEndParams prm) {
    grid_dep_launch();
    grid_dep_wait();
    const int block = blockIdx.x, sums = prm.of[kMlpSums - 1].blocks;
    if (block < sums) {
        const int which = (block >= prm.of[0].blocks) + (block >= prm.of[1].blocks);
        const MlpReduce &w = prm.of[which];
        const int quads = (w.cols + 3) / 4;
        const long long i = (long long)(block - (which ? prm.of[which - 1].blocks : 0)) * 256 + threadIdx.x;
        if (i >= (long long)w.rows * quads) return;
        const long long r = i / quads;
        const int c = (int)(i - r * quads) * 4, n = min(4, w.cols - c);
        const float *p = w.partial + r * w.stride + c;
        float4 s = *reinterpret_cast<const float4 *>(p);
        for (int k = 1; k < w.splits; ++k) {
            const float4 v = *reinterpret_cast<const float4 *>(p + k * w.split_stride);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        float v[4] = {s.x, s.y, s.z, s.w};
        if (w.bias != nullptr)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) v[e] += __bfloat162float(w.bias[c + e]);
        if (w.side != nullptr)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) v[e] += __bfloat162float(w.side[r * w.side_stride + c + e]);
        __nv_bfloat16 *out = w.out + r * w.out_stride + c;
        if (w.vec && n == 4) {
            *reinterpret_cast<uint2 *>(out) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) out[e] = __float2bfloat16_rn(v[e]);
        }
        return;
    }
    __shared__ float part[8][32];
    const bool second = block >= prm.bias_blocks;
    const MlpSum &b = prm.bias[second];
    const int lane = threadIdx.x % 32, g = threadIdx.x / 32, c = (block - (second ? prm.bias_blocks : sums)) * 32 + lane;
    float s = 0.0f;
    if (c < b.total)
#pragma unroll 4
        for (int k = g; k < prm.stretches; k += 8) s += b.partial[(long long)k * b.total + c];
    part[g][lane] = s;
    __syncthreads();
    if (g == 0 && c < b.total) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += part[i][lane];
        b.out[c] = __float2bfloat16_rn(s);
    }
}

}  // namespace kla
