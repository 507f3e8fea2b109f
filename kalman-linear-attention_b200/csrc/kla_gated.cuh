// The gated recurrence, forward, backward and one token:
//
//   z_t = sigmoid(-g_t),  a_t = 1 - z_t = sigmoid(g_t);   h_t = a_t h_{t-1} + z_t x_t,   h_{-1} = the state a sequence starts from
//   c_t = dh_t + u_{t+1},  u_t = a_t c_t,  u after the last step = the gradient of the state it leaves;
//   dx_t = z_t c_t,   dg_t = c_t (h_{t-1} - x_t) z_t a_t,   gradient of the starting state = u_0
//
// Every channel of every sequence is a chain of its own, and over a stretch of steps both recurrences are affine maps with the
// same slope A = prod a_t: h -> A h + F and u -> A u + R. A step is taken as h - z h + z x with two fused operations: what is
// rounded is then small beside 1 - a where a gate holds the state for thousands of steps, which a = 1 - z rounded is not.
//
// A CTA owns 64 channels of one sequence and walks it in tiles of kGatedWarps x TS steps. Each warp takes TS consecutive steps
// of the tile, each lane two channels. The warp's rows come in by asynchronous copies into a ring of its own in shared memory,
// tiles ahead, so that what is in flight (64 KB an SM and more) does not hang on registers or on other warps; it composes the map
// of its steps, puts it in shared memory, and after one barrier folds the maps of the warps in front of it to get its own first
// state; then it walks its steps once more and stores. So every input is read and every output written once. The backward needs the states in front of its steps: the forward leaves one per
// kGatedUnit steps and channel, and the backward, whose tile is one such unit, walks forward from it in registers, which is
// 4 bytes per 64 steps to read in place of h.
// With a cluster of CTAs a sequence's tiles go round robin to its CTAs, which exchange their tiles' maps through distributed
// shared memory once a round: the way to fill the GPU with few sequences or channels.
#pragma once

#include <type_traits>

#include "kla_common.cuh"

namespace kla {

constexpr int kGatedWarps = 8;
constexpr int kGatedChannels = 64;  // of a CTA
constexpr int kGatedUnit = 64;      // steps between the states the forward leaves for the backward
constexpr int kGatedMaxCluster = 8;

struct GatedParams {
    int N, L, D;        // sequences, rows of a batch entry (packed: of all sequences), channels
    int blocks;         // channel blocks
    Tensor3 x, g, h;
    int x_width, g_width, dh_width;  // bytes a copy of their rows may move (gated_fetch)
    const int *cu;      // [N + 1] bounds of packed sequences or nullptr: sequences are batch entries
    const float *h0;    // [N, D] or nullptr: zeros
    float *end;         // [N, D]
    float *ckpt;        // states the backward starts from, or nullptr
    Tensor3 dh, dx, dg;
    const float *dend;  // [N, D] or nullptr: zeros
    float *dh0;         // [N, D] or nullptr
};

// A lane's two channels: neighbours where every row can be written in pairs (PAIR), otherwise 32 apart.
template <bool PAIR>
struct Lane {
    int lane, c0, c1;  // its channels within the tensor
    bool on0, on1;     // whether they exist
    __device__ __forceinline__ Lane(int block, int lane_, int D) : lane(lane_) {
        c0 = block * kGatedChannels + (PAIR ? 2 * lane : lane);
        c1 = PAIR ? c0 + 1 : c0 + 32;
        on0 = c0 < D;
        on1 = c1 < D;
    }
    // from a row of the block's 64 channels in shared memory
    __device__ __forceinline__ float2 take(const float *row) const { return PAIR ? *reinterpret_cast<const float2 *>(row + 2 * lane) : make_float2(row[lane], row[lane + 32]); }
    __device__ __forceinline__ float2 take(const __nv_bfloat16 *row) const {
        if constexpr (PAIR) {
            const uint32_t v = *reinterpret_cast<const uint32_t *>(row + 2 * lane);
            return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
        } else {
            return make_float2(__bfloat162float(row[lane]), __bfloat162float(row[lane + 32]));
        }
    }
    __device__ __forceinline__ void store(float *row, float2 y) const {
        if constexpr (PAIR) {
            if (on0) *reinterpret_cast<float2 *>(row + c0) = y;
        } else {
            if (on0) row[c0] = y.x;
            if (on1) row[c1] = y.y;
        }
    }
    __device__ __forceinline__ void store(__nv_bfloat16 *row, float2 y) const {
        const __nv_bfloat162 v = __floats2bfloat162_rn(y.x, y.y);
        if constexpr (PAIR) {
            if (on0) *reinterpret_cast<__nv_bfloat162 *>(row + c0) = v;
        } else {
            if (on0) row[c0] = __low2bfloat16(v);
            if (on1) row[c1] = __high2bfloat16(v);
        }
    }
    // states are rows of their own alignment: one by one
    __device__ __forceinline__ float2 load_state(const float *row) const { return make_float2(on0 ? row[c0] : 0.0f, on1 ? row[c1] : 0.0f); }
    __device__ __forceinline__ void store_state(float *row, float2 y) const {
        if (on0) row[c0] = y.x;
        if (on1) row[c1] = y.y;
    }
};

__device__ __forceinline__ void gated_copy(void *dst, const void *src, int bytes, bool sixteen) {
    if (sixteen) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
// `rows` (of TS at most) rows of the block's 64 channels into shared memory by one warp. width: bytes a copy moves, as far as
// the tensor's alignment goes (16 or 4; bfloat16 rows at odd places have 2 and are loaded and stored one by one). Channels past
// the tensor's are zeros.
template <typename T, int TS>
__device__ __forceinline__ void gated_fetch(T *dst, const T *src, long long stride, int rows, int block, int D, int width, int lane) {
    const int c_block = block * kGatedChannels;
    src += c_block;
    if (width >= 4) {
        const bool sixteen = width == 16;
        const int per = (sixteen ? 16 : 4) / (int)sizeof(T), pieces = kGatedChannels / per;
        constexpr int kFirst = 32 / (kGatedChannels * (int)sizeof(T) / 16);  // rows that 32 pieces of 16 bytes are
        if (sixteen) {
            const int c = lane % pieces * per;
            const int bytes = max(0, min(16, (D - c_block - c) * (int)sizeof(T)));
            const T *from = bytes > 0 ? src + c : src;
#pragma unroll
            for (int i = 0; i < TS; i += kFirst) {
                const int r = i + lane / pieces;
                if (r < rows) gated_copy(dst + r * kGatedChannels + c, from + r * stride, bytes, true);
            }
        } else {
#pragma unroll
            for (int h = 0; h < kGatedChannels * (int)sizeof(T) / 128; ++h) {
                const int c = (lane + 32 * h) * per;
                const int bytes = c_block + c < D ? 4 : 0;  // (pairs of bfloat16: D is even)
                const T *from = bytes > 0 ? src + c : src;
#pragma unroll
                for (int r = 0; r < TS; ++r)
                    if (r < rows) gated_copy(dst + r * kGatedChannels + c, from + r * stride, bytes, false);
            }
        }
    } else {
        const int n0 = c_block + lane < D, n1 = c_block + lane + 32 < D;
#pragma unroll
        for (int r0 = 0; r0 < TS; r0 += 8) {
            T a[8], b[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                a[r] = b[r] = from_f32<T>(0.0f);
                if (r0 + r < rows) {
                    if (n0) a[r] = src[(r0 + r) * stride + lane];
                    if (n1) b[r] = src[(r0 + r) * stride + lane + 32];
                }
            }
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r0 + r < rows) {
                    dst[(r0 + r) * kGatedChannels + lane] = a[r];
                    dst[(r0 + r) * kGatedChannels + lane + 32] = b[r];
                }
        }
    }
}
__device__ __forceinline__ void gated_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void gated_arrived() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    __syncwarp();
}

// Steps of a warp and tiles of its ring, so that two CTAs' rings fit an SM.
template <typename T>
struct GatedFwdShape {
    static constexpr int TS = sizeof(T) == 2 ? 16 : 8, S = 3;
    static constexpr size_t kBytes = (size_t)kGatedWarps * S * 2 * TS * kGatedChannels * sizeof(T);
};
template <typename T>
struct GatedBwdShape {
    static constexpr int TS = kGatedUnit / kGatedWarps, S = sizeof(T) == 2 ? 3 : 2;
    static constexpr size_t kBytes = (size_t)kGatedWarps * S * 3 * TS * kGatedChannels * sizeof(T);
};

// The rows a CTA's sequence covers. Bounds of packed sequences come from the device unseen by the host: clamped, so that no
// value of theirs leads out of the tensors.
struct GatedSpan {
    int b, lo, len, unit;  // batch entry, first row, rows, first unit
};
__device__ __forceinline__ GatedSpan gated_span(const GatedParams &p, int n) {
    if (p.cu == nullptr) return GatedSpan{n, 0, p.L, n * ((p.L + kGatedUnit - 1) / kGatedUnit)};
    const int lo = min(max(p.cu[n], 0), p.L), hi = min(max(p.cu[n + 1], lo), p.L);
    return GatedSpan{0, lo, hi - lo, lo / kGatedUnit + n};
}
template <typename T>
__device__ __forceinline__ T *gated_rows(const Tensor3 &t, const GatedSpan &s) {
    return static_cast<T *>(const_cast<void *>(t.ptr)) + (long long)s.b * t.sb + (long long)s.lo * t.st;
}

// Rows in front of the first and behind the last packed sequence belong to none: zeros.
template <typename T, bool PAIR>
__device__ __forceinline__ void gated_clear(const GatedParams &p, const Tensor3 &t, const Lane<PAIR> &ln, int warp, int rank, int ranks) {
    const int first = min(max(p.cu[0], 0), p.L), last = min(max(p.cu[p.N], 0), p.L);
    for (int r = rank * kGatedWarps + warp; r < p.L; r += ranks * kGatedWarps)
        if (r < first || r >= last) ln.store(static_cast<T *>(const_cast<void *>(t.ptr)) + (long long)r * t.st, make_float2(0.0f, 0.0f));
}

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// -z of a gate: a gate of +-inf gives exactly 0 or -1
__device__ __forceinline__ float2 neg_z(float2 g) {
    return make_float2(rcp_approx(-1.0f - ex2_approx(g.x * kLog2e)), rcp_approx(-1.0f - ex2_approx(g.y * kLog2e)));
}
// -z and z a, both with the relative accuracy of the smaller of z and a
__device__ __forceinline__ void neg_z_slope(float g, float &nz, float &za) {
    const float e = ex2_approx(-fabsf(g) * kLog2e), r = rcp_approx(1.0f + e), small = e * r;
    nz = g >= 0.0f ? -small : -r;
    za = small * r;
}

// h -> A h + F of a stretch, two channels
struct Map2 {
    float2 A, F;
    __device__ __forceinline__ float2 operator()(float2 h) const { return fma2(A, h, F); }
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a 16-byte store into another CTA of the cluster, at the place `here` has in this one
__device__ __forceinline__ void cluster_store(const void *here, uint32_t rank, float4 v) {
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_u32(here)), "r"(rank));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// Maps of the CTA's warps and (CLUSTER) of the cluster's CTAs, twice: a round writes one copy while the slowest reader of the
// round before may still be in the other.
template <bool CLUSTER>
struct GatedShared {
    float4 warp[2][kGatedWarps][32];
    float4 cta[2][CLUSTER ? kGatedMaxCluster : 1][32];
    float2 carry[2][32];
};

// Called by all threads with the map of the warp's own steps: the value in front of the warp's steps. The value in front of the round is
// sh.carry[buf] (for the first round put there by the warp that is last in the fold), the one behind it goes to the other copy.
// REVERSE: values come from behind. One barrier of the CTA, with CLUSTER one of the cluster.
template <bool CLUSTER, bool REVERSE>
__device__ __forceinline__ float2 gated_exchange(GatedShared<CLUSTER> &sh, int buf, Map2 own, int warp, int lane, int rank, int ranks) {
    auto map = [](const float4 &v) { return Map2{make_float2(v.x, v.y), make_float2(v.z, v.w)}; };
    const int place = REVERSE ? kGatedWarps - 1 - warp : warp;  // in the order of the fold
    sh.warp[buf][place][lane] = make_float4(own.A.x, own.A.y, own.F.x, own.F.y);
    __syncthreads();
    float2 mine;
    if constexpr (CLUSTER) {
        if (warp == 0) {  // the CTA's map to all
            Map2 all{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int i = 0; i < kGatedWarps; ++i) {
                const Map2 m = map(sh.warp[buf][i][lane]);
                all.F = m(all.F);
                all.A = mul2(m.A, all.A);
            }
            const float4 v = make_float4(all.A.x, all.A.y, all.F.x, all.F.y);
            for (int r = 0; r < ranks; ++r) cluster_store(&sh.cta[buf][rank][lane], r, v);
        }
        cluster_sync();
        mine = sh.carry[buf][lane];
        const int before = REVERSE ? ranks - 1 - rank : rank;
        for (int i = 0; i < before; ++i) mine = map(sh.cta[buf][REVERSE ? ranks - 1 - i : i][lane])(mine);
        if (place == kGatedWarps - 1) {  // (the warp that folds most anyway)
            float2 end = mine;
            for (int i = before; i < ranks; ++i) end = map(sh.cta[buf][REVERSE ? ranks - 1 - i : i][lane])(end);
            sh.carry[buf ^ 1][lane] = end;
        }
    } else {
        mine = sh.carry[buf][lane];
    }
#pragma unroll
    for (int i = 0; i < kGatedWarps - 1; ++i)
        if (i < place) mine = map(sh.warp[buf][i][lane])(mine);
    if (!CLUSTER && place == kGatedWarps - 1) sh.carry[buf ^ 1][lane] = own(mine);
    return mine;
}

// Grid: sequences x channel blocks x cluster, the last fastest; with packed sequences one sequence more, which clears the rows
// that belong to none.
template <typename T, bool PAIR, bool CLUSTER>
__global__ void __launch_bounds__(kGatedWarps * 32, 2) kla_gated_fwd_kernel(const __grid_constant__ GatedParams prm) {
    using Shape = GatedFwdShape<T>;
    constexpr int TS = Shape::TS, S = Shape::S, TT = kGatedWarps * TS;
    __shared__ GatedShared<CLUSTER> sh;
    extern __shared__ __align__(16) unsigned char ring_bytes[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = CLUSTER ? (int)cluster_rank() : 0, ranks = CLUSTER ? (int)cluster_size() : 1;
    const int cell = blockIdx.x / ranks, n = cell / prm.blocks, block = cell % prm.blocks;
    const Lane<PAIR> ln(block, lane, prm.D);
    if (n == prm.N) return gated_clear<T, PAIR>(prm, prm.h, ln, warp, rank, ranks);  // the whole cluster returns
    if constexpr (CLUSTER) cluster_sync();  // every CTA has begun: its shared memory may be written
    const GatedSpan span = gated_span(prm, n);
    const T *x = gated_rows<const T>(prm.x, span), *g = gated_rows<const T>(prm.g, span);
    T *h_out = gated_rows<T>(prm.h, span);
    T *ring = reinterpret_cast<T *>(ring_bytes) + warp * S * 2 * TS * kGatedChannels;
    const int rounds = (span.len + TT * ranks - 1) / (TT * ranks), len = span.len;
    if (warp == kGatedWarps - 1) sh.carry[0][lane] = prm.h0 ? ln.load_state(prm.h0 + (long long)n * prm.D) : make_float2(0.0f, 0.0f);

    int fetched = 0, slot_in = 0;
    auto fetch = [&] {  // the next round's rows, where there is one; a group of copies either way
        if (fetched < rounds) {
            const int t0 = (fetched * ranks + rank) * TT + warp * TS, rows = len - t0;
            T *to = ring + slot_in * 2 * TS * kGatedChannels;
            gated_fetch<T, TS>(to, g + (long long)t0 * prm.g.st, prm.g.st, rows, block, prm.D, prm.g_width, lane);
            gated_fetch<T, TS>(to + TS * kGatedChannels, x + (long long)t0 * prm.x.st, prm.x.st, rows, block, prm.D, prm.x_width, lane);
        }
        gated_commit();
        ++fetched;
        if (++slot_in == S) slot_in = 0;
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) fetch();
    int slot = 0;
    for (int round = 0; round < rounds; ++round) {
        const int t0 = (round * ranks + rank) * TT + warp * TS, cnt = len - t0;
        gated_arrived<S - 2>();
        fetch();  // over the round before
        const T *gs = ring + slot * 2 * TS * kGatedChannels, *xs = gs + TS * kGatedChannels;
        if (++slot == S) slot = 0;
        float2 nz[TS];
        Map2 own{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
        auto compose = [&](int i) {
            nz[i] = neg_z(ln.take(gs + i * kGatedChannels));
            own.A = fma2(nz[i], own.A, own.A);
            own.F = fma2(nz[i], neg2(ln.take(xs + i * kGatedChannels)), fma2(nz[i], own.F, own.F));
        };
        if (cnt >= TS) {
#pragma unroll
            for (int i = 0; i < TS; ++i) compose(i);
        } else {
#pragma unroll
            for (int i = 0; i < TS; ++i)
                if (i < cnt) compose(i);
        }
        float2 h = gated_exchange<CLUSTER, false>(sh, round & 1, own, warp, lane, rank, ranks);
        if (prm.ckpt != nullptr && t0 % kGatedUnit == 0 && cnt > 0)
            ln.store_state(prm.ckpt + (long long)(span.unit + t0 / kGatedUnit) * prm.D, h);
        T *to = h_out + (long long)t0 * prm.h.st;
        auto walk = [&](int i) {
            h = fma2(nz[i], neg2(ln.take(xs + i * kGatedChannels)), fma2(nz[i], h, h));
            ln.store(to, h);
            to += prm.h.st;
        };
        if (cnt >= TS) {
#pragma unroll
            for (int i = 0; i < TS; ++i) walk(i);
        } else {
#pragma unroll
            for (int i = 0; i < TS; ++i)
                if (i < cnt) walk(i);
        }
    }
    if (warp == kGatedWarps - 1 && rank == 0) ln.store_state(prm.end + (long long)n * prm.D, sh.carry[rounds & 1][lane]);  // its own
}

template <typename T, bool PAIR, bool CLUSTER>
__global__ void __launch_bounds__(kGatedWarps * 32, 2) kla_gated_bwd_kernel(const __grid_constant__ GatedParams prm) {
    using Shape = GatedBwdShape<T>;
    constexpr int TS = Shape::TS, S = Shape::S, kTile = TS * kGatedChannels;
    __shared__ GatedShared<CLUSTER> sh;
    __shared__ float4 fw[2][kGatedWarps][32];  // maps of the warps forwards
    extern __shared__ __align__(16) unsigned char ring_bytes[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = CLUSTER ? (int)cluster_rank() : 0, ranks = CLUSTER ? (int)cluster_size() : 1;
    const int cell = blockIdx.x / ranks, n = cell / prm.blocks, block = cell % prm.blocks;
    const Lane<PAIR> ln(block, lane, prm.D);
    if (n == prm.N) {
        gated_clear<T, PAIR>(prm, prm.dx, ln, warp, rank, ranks);
        return gated_clear<T, PAIR>(prm, prm.dg, ln, warp, rank, ranks);
    }
    if constexpr (CLUSTER) cluster_sync();
    const GatedSpan span = gated_span(prm, n);
    const T *x = gated_rows<const T>(prm.x, span), *g = gated_rows<const T>(prm.g, span), *dh = gated_rows<const T>(prm.dh, span);
    T *dx = gated_rows<T>(prm.dx, span), *dg = gated_rows<T>(prm.dg, span);
    T *ring = reinterpret_cast<T *>(ring_bytes) + warp * S * 3 * kTile;
    const int len = span.len, rounds = (len + kGatedUnit * ranks - 1) / (kGatedUnit * ranks);
    // copies of the exchange by parity of the rounds done
    if (warp == 0) sh.carry[0][lane] = prm.dend ? ln.load_state(prm.dend + (long long)n * prm.D) : make_float2(0.0f, 0.0f);

    int fetched = rounds - 1, slot_in = 0;
    auto fetch = [&] {  // rounds from the last one on
        if (fetched >= 0) {
            const int t0 = (fetched * ranks + rank) * kGatedUnit + warp * TS, rows = len - t0;
            T *to = ring + slot_in * 3 * kTile;
            gated_fetch<T, TS>(to, g + (long long)t0 * prm.g.st, prm.g.st, rows, block, prm.D, prm.g_width, lane);
            gated_fetch<T, TS>(to + kTile, x + (long long)t0 * prm.x.st, prm.x.st, rows, block, prm.D, prm.x_width, lane);
            gated_fetch<T, TS>(to + 2 * kTile, dh + (long long)t0 * prm.dh.st, prm.dh.st, rows, block, prm.D, prm.dh_width, lane);
        }
        gated_commit();
        --fetched;
        if (++slot_in == S) slot_in = 0;
    };
    // the state in front of a round's unit
    auto front = [&](int round) {
        const int unit = round * ranks + rank;
        return round >= 0 && unit * kGatedUnit < len ? ln.load_state(prm.ckpt + (long long)(span.unit + unit) * prm.D) : make_float2(0.0f, 0.0f);
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) fetch();
    float2 next = front(rounds - 1);
    int slot = 0;
    for (int round = rounds - 1; round >= 0; --round) {
        const int t0 = (round * ranks + rank) * kGatedUnit + warp * TS, cnt = len - t0, buf = (rounds - 1 - round) & 1;
        float2 h = next;
        next = front(round - 1);
        gated_arrived<S - 2>();
        fetch();
        const T *gs = ring + slot * 3 * kTile, *xs = gs + kTile, *ds = xs + kTile;
        if (++slot == S) slot = 0;
        float2 nz[TS], za[TS];
        Map2 back{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
        float2 F = make_float2(0.0f, 0.0f);
        auto compose = [&](auto full) {
            constexpr bool FULL = decltype(full)::value;
#pragma unroll
            for (int i = 0; i < TS; ++i)
                if (FULL || i < cnt) {
                    const float2 gi = ln.take(gs + i * kGatedChannels);
                    neg_z_slope(gi.x, nz[i].x, za[i].x);
                    neg_z_slope(gi.y, nz[i].y, za[i].y);
                    back.A = fma2(nz[i], back.A, back.A);
                    F = fma2(nz[i], neg2(ln.take(xs + i * kGatedChannels)), fma2(nz[i], F, F));
                }
#pragma unroll
            for (int i = TS - 1; i >= 0; --i)
                if (FULL || i < cnt) {
                    const float2 ci = add2(ln.take(ds + i * kGatedChannels), back.F);
                    back.F = fma2(nz[i], ci, ci);
                }
        };
        if (cnt >= TS) compose(std::true_type{});
        else compose(std::false_type{});
        fw[buf][warp][lane] = make_float4(back.A.x, back.A.y, F.x, F.y);
        float2 u = gated_exchange<CLUSTER, true>(sh, buf, back, warp, lane, rank, ranks);
        for (int w = 0; w < warp; ++w) {
            const float4 m = fw[buf][w][lane];
            h = fma2(make_float2(m.x, m.y), h, make_float2(m.z, m.w));
        }
        auto walk = [&](auto full) {
            constexpr bool FULL = decltype(full)::value;
            float2 c[TS];
#pragma unroll
            for (int i = TS - 1; i >= 0; --i)
                if (FULL || i < cnt) {
                    c[i] = add2(ln.take(ds + i * kGatedChannels), u);
                    u = fma2(nz[i], c[i], c[i]);
                }
            T *to_x = dx + (long long)t0 * prm.dx.st, *to_g = dg + (long long)t0 * prm.dg.st;
#pragma unroll
            for (int i = 0; i < TS; ++i)
                if (FULL || i < cnt) {
                    const float2 nx = neg2(ln.take(xs + i * kGatedChannels));
                    ln.store(to_x + i * prm.dx.st, mul2(neg2(nz[i]), c[i]));
                    ln.store(to_g + i * prm.dg.st, mul2(mul2(za[i], c[i]), add2(h, nx)));
                    h = fma2(nz[i], nx, fma2(nz[i], h, h));
                }
        };
        if (cnt >= TS) walk(std::true_type{});
        else walk(std::false_type{});
    }
    if (prm.dh0 != nullptr && warp == 0 && rank == 0) ln.store_state(prm.dh0 + (long long)n * prm.D, sh.carry[rounds & 1][lane]);  // its own
}

// One token: rows [B, D] of x and g, the state read and written as float32 (in place where both are the same).
struct GatedStepParams {
    long long n;  // B * D
    int D;
    const void *x, *g;
    long long x_sb, g_sb;
    const float *state;
    float *state_out;
    void *h;
};
template <typename T>
__global__ void __launch_bounds__(256) kla_gated_step_kernel(const GatedStepParams prm) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= prm.n) return;
    const long long b = i / prm.D;
    const int d = (int)(i - b * prm.D);
    const float x = to_f32<T>(static_cast<const T *>(prm.x)[b * prm.x_sb + d]);
    const float nz = rcp_approx(-1.0f - ex2_approx(to_f32<T>(static_cast<const T *>(prm.g)[b * prm.g_sb + d]) * kLog2e));
    const float s = prm.state[i], h = fmaf(nz, -x, fmaf(nz, s, s));
    prm.state_out[i] = h;
    static_cast<T *>(prm.h)[i] = from_f32<T>(h);
}

}  // namespace kla
