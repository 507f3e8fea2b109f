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
// of the tile, each lane two channels: it loads its share of x and g straight into registers (one 128-byte row of bfloat16 a
// warp access) a tile ahead, composes the map of its steps, puts it in shared memory, and after one barrier folds the maps of
// the warps in front of it to get its own first state; then it walks its steps once more and stores. So every input is read
// and every output written once. The backward needs the states in front of its steps: the forward leaves one per
// kGatedUnit steps and channel, and the backward, whose tile is one such unit, walks forward from it in registers, which is
// 4 bytes per 64 steps to read in place of h.
// With a cluster of CTAs a sequence's tiles go round robin to its CTAs, which exchange their tiles' maps through distributed
// shared memory once a round: the way to fill the GPU with few sequences or channels.
#pragma once

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
    const int *cu;      // [N + 1] bounds of packed sequences or nullptr: sequences are batch entries
    const float *h0;    // [N, D] or nullptr: zeros
    float *end;         // [N, D]
    float *ckpt;        // states the backward starts from, or nullptr
    Tensor3 dh, dx, dg;
    const float *dend;  // [N, D] or nullptr: zeros
    float *dh0;         // [N, D] or nullptr
};

// Two channels of one row as they lie in memory. PAIR: neighbouring ones by one access (rows allow it); otherwise channels 32
// apart, one by one, each where it exists.
template <typename T>
struct Two;
template <>
struct Two<float> {
    float a, b;
    __device__ __forceinline__ float2 wide() const { return make_float2(a, b); }
};
template <>
struct Two<__nv_bfloat16> {
    uint32_t v;  // low half: the first channel
    __device__ __forceinline__ float2 wide() const { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
};

template <bool PAIR>
struct Lane {
    int c0, c1;     // its channels within the tensor
    bool on0, on1;  // whether they exist
    __device__ __forceinline__ Lane(int block, int lane, int D) {
        c0 = block * kGatedChannels + (PAIR ? 2 * lane : lane);
        c1 = PAIR ? c0 + 1 : c0 + 32;
        on0 = c0 < D;
        on1 = c1 < D;
    }
    __device__ __forceinline__ Two<float> load(const float *row) const {
        Two<float> r{0.0f, 0.0f};
        if constexpr (PAIR) {
            if (on0) asm volatile("ld.global.nc.L1::no_allocate.v2.f32 {%0, %1}, [%2];" : "=f"(r.a), "=f"(r.b) : "l"(row + c0));
        } else {
            if (on0) r.a = __ldg(row + c0);
            if (on1) r.b = __ldg(row + c1);
        }
        return r;
    }
    __device__ __forceinline__ Two<__nv_bfloat16> load(const __nv_bfloat16 *row) const {
        Two<__nv_bfloat16> r{0u};
        if constexpr (PAIR) {
            if (on0) asm volatile("ld.global.nc.L1::no_allocate.b32 %0, [%1];" : "=r"(r.v) : "l"(row + c0));
        } else {
            const unsigned short *p = reinterpret_cast<const unsigned short *>(row);
            const uint32_t lo = on0 ? __ldg(p + c0) : 0u, hi = on1 ? __ldg(p + c1) : 0u;
            r.v = lo | hi << 16;
        }
        return r;
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
};

// Called by all threads with the map of the warp's own steps: the value in front of the warp's steps, and `carry` moved past the
// whole round (a tile of every CTA). REVERSE: values come from behind. One barrier of the CTA, with CLUSTER one of the cluster.
template <bool CLUSTER, bool REVERSE>
__device__ __forceinline__ float2 gated_exchange(GatedShared<CLUSTER> &sh, int buf, Map2 own, float2 &carry, int warp, int lane, int rank, int ranks) {
    auto map = [](const float4 &v) { return Map2{make_float2(v.x, v.y), make_float2(v.z, v.w)}; };
    sh.warp[buf][warp][lane] = make_float4(own.A.x, own.A.y, own.F.x, own.F.y);
    __syncthreads();
    if constexpr (CLUSTER) {
        if (warp < ranks) {  // warp r takes the CTA's map to rank r
            Map2 all{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int i = 0; i < kGatedWarps; ++i) {
                const Map2 m = map(sh.warp[buf][REVERSE ? kGatedWarps - 1 - i : i][lane]);
                all.F = m(all.F);
                all.A = mul2(m.A, all.A);
            }
            cluster_store(&sh.cta[buf][rank][lane], warp, make_float4(all.A.x, all.A.y, all.F.x, all.F.y));
        }
        cluster_sync();
        float2 mine = carry;
        for (int i = 0; i < ranks; ++i) {
            const int r = REVERSE ? ranks - 1 - i : i;
            if (r == rank) mine = carry;
            carry = map(sh.cta[buf][r][lane])(carry);
        }
        for (int i = 0; i < kGatedWarps - 1; ++i) {
            const int w = REVERSE ? kGatedWarps - 1 - i : i;
            if (REVERSE ? w <= warp : w >= warp) break;
            mine = map(sh.warp[buf][w][lane])(mine);
        }
        return mine;
    } else {
        float2 mine = carry;
#pragma unroll
        for (int i = 0; i < kGatedWarps; ++i) {
            const int w = REVERSE ? kGatedWarps - 1 - i : i;
            if (w == warp) mine = carry;
            carry = map(sh.warp[buf][w][lane])(carry);
        }
        return mine;
    }
}

// Grid: sequences x channel blocks x cluster, the last fastest; with packed sequences one sequence more, which clears the rows
// that belong to none.
template <typename T, bool PAIR, bool CLUSTER, int TS>
__global__ void __launch_bounds__(kGatedWarps * 32) kla_gated_fwd_kernel(const __grid_constant__ GatedParams prm) {
    __shared__ GatedShared<CLUSTER> sh;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = CLUSTER ? (int)cluster_rank() : 0, ranks = CLUSTER ? (int)cluster_size() : 1;
    const int cell = blockIdx.x / ranks, n = cell / prm.blocks;
    const Lane<PAIR> ln(cell % prm.blocks, lane, prm.D);
    if (n == prm.N) return gated_clear<T, PAIR>(prm, prm.h, ln, warp, rank, ranks);  // the whole cluster returns
    if constexpr (CLUSTER) cluster_sync();  // every CTA has begun: its shared memory may be written
    const GatedSpan span = gated_span(prm, n);
    const T *x = gated_rows<const T>(prm.x, span), *g = gated_rows<const T>(prm.g, span);
    T *h_out = gated_rows<T>(prm.h, span);
    constexpr int TT = kGatedWarps * TS;
    const int rounds = (span.len + TT * ranks - 1) / (TT * ranks);
    float2 carry = prm.h0 ? ln.load_state(prm.h0 + (long long)n * prm.D) : make_float2(0.0f, 0.0f);

    Two<T> xr[TS], gr[TS], xn[TS], gn[TS];
    auto fetch = [&](int round) {
        const int t0 = (round * ranks + rank) * TT + warp * TS, cnt = span.len - t0;
#pragma unroll
        for (int i = 0; i < TS; ++i)
            if (i < cnt) {
                gn[i] = ln.load(g + (long long)(t0 + i) * prm.g.st);
                xn[i] = ln.load(x + (long long)(t0 + i) * prm.x.st);
            }
    };
    fetch(0);
    for (int round = 0; round < rounds; ++round) {
        const int t0 = (round * ranks + rank) * TT + warp * TS, cnt = span.len - t0;
#pragma unroll
        for (int i = 0; i < TS; ++i) { xr[i] = xn[i]; gr[i] = gn[i]; }
        if (round + 1 < rounds) fetch(round + 1);
        float2 nz[TS];
        Map2 own{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int i = 0; i < TS; ++i)
            if (i < cnt) {
                nz[i] = neg_z(gr[i].wide());
                own.A = fma2(nz[i], own.A, own.A);
                own.F = fma2(nz[i], neg2(xr[i].wide()), fma2(nz[i], own.F, own.F));
            }
        float2 h = gated_exchange<CLUSTER, false>(sh, round & 1, own, carry, warp, lane, rank, ranks);
        if (prm.ckpt != nullptr && t0 % kGatedUnit == 0 && cnt > 0)
            ln.store_state(prm.ckpt + (long long)(span.unit + t0 / kGatedUnit) * prm.D, h);
#pragma unroll
        for (int i = 0; i < TS; ++i)
            if (i < cnt) {
                h = fma2(nz[i], neg2(xr[i].wide()), fma2(nz[i], h, h));
                ln.store(h_out + (long long)(t0 + i) * prm.h.st, h);
            }
    }
    if (warp == 0 && rank == 0) ln.store_state(prm.end + (long long)n * prm.D, carry);
}

template <typename T, bool PAIR, bool CLUSTER>
__global__ void __launch_bounds__(kGatedWarps * 32) kla_gated_bwd_kernel(const __grid_constant__ GatedParams prm) {
    constexpr int TS = kGatedUnit / kGatedWarps;
    __shared__ GatedShared<CLUSTER> sh;
    __shared__ float4 fw[2][kGatedWarps][32];  // maps of the warps forwards
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = CLUSTER ? (int)cluster_rank() : 0, ranks = CLUSTER ? (int)cluster_size() : 1;
    const int cell = blockIdx.x / ranks, n = cell / prm.blocks;
    const Lane<PAIR> ln(cell % prm.blocks, lane, prm.D);
    if (n == prm.N) {
        gated_clear<T, PAIR>(prm, prm.dx, ln, warp, rank, ranks);
        return gated_clear<T, PAIR>(prm, prm.dg, ln, warp, rank, ranks);
    }
    if constexpr (CLUSTER) cluster_sync();
    const GatedSpan span = gated_span(prm, n);
    const T *x = gated_rows<const T>(prm.x, span), *g = gated_rows<const T>(prm.g, span), *dh = gated_rows<const T>(prm.dh, span);
    T *dx = gated_rows<T>(prm.dx, span), *dg = gated_rows<T>(prm.dg, span);
    const int rounds = (span.len + kGatedUnit * ranks - 1) / (kGatedUnit * ranks);
    float2 carry = prm.dend ? ln.load_state(prm.dend + (long long)n * prm.D) : make_float2(0.0f, 0.0f);

    Two<T> xr[TS], gr[TS], dr[TS], xn[TS], gn[TS], dn[TS];
    float2 first, first_next = make_float2(0.0f, 0.0f);
    auto fetch = [&](int round) {
        const int unit = round * ranks + rank, t0 = unit * kGatedUnit + warp * TS, cnt = span.len - t0;
#pragma unroll
        for (int i = 0; i < TS; ++i)
            if (i < cnt) {
                gn[i] = ln.load(g + (long long)(t0 + i) * prm.g.st);
                dn[i] = ln.load(dh + (long long)(t0 + i) * prm.dh.st);
                xn[i] = ln.load(x + (long long)(t0 + i) * prm.x.st);
            }
        if (unit * kGatedUnit < span.len) first_next = ln.load_state(prm.ckpt + (long long)(span.unit + unit) * prm.D);
    };
    if (rounds > 0) fetch(rounds - 1);
    for (int round = rounds - 1; round >= 0; --round) {
        const int t0 = (round * ranks + rank) * kGatedUnit + warp * TS, cnt = span.len - t0, buf = round & 1;
#pragma unroll
        for (int i = 0; i < TS; ++i) { xr[i] = xn[i]; gr[i] = gn[i]; dr[i] = dn[i]; }
        first = first_next;
        if (round > 0) fetch(round - 1);
        float2 nz[TS], za[TS], c[TS];
        Map2 back{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
        float2 F = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < TS; ++i)
            if (i < cnt) {
                const float2 gi = gr[i].wide();
                neg_z_slope(gi.x, nz[i].x, za[i].x);
                neg_z_slope(gi.y, nz[i].y, za[i].y);
                back.A = fma2(nz[i], back.A, back.A);
                F = fma2(nz[i], neg2(xr[i].wide()), fma2(nz[i], F, F));
            }
#pragma unroll
        for (int i = TS - 1; i >= 0; --i)
            if (i < cnt) {
                const float2 ci = add2(dr[i].wide(), back.F);
                back.F = fma2(nz[i], ci, ci);
            }
        fw[buf][warp][lane] = make_float4(back.A.x, back.A.y, F.x, F.y);
        float2 u = gated_exchange<CLUSTER, true>(sh, buf, back, carry, warp, lane, rank, ranks);
        float2 h = first;
        for (int w = 0; w < warp; ++w) {
            const float4 m = fw[buf][w][lane];
            h = fma2(make_float2(m.x, m.y), h, make_float2(m.z, m.w));
        }
#pragma unroll
        for (int i = TS - 1; i >= 0; --i)
            if (i < cnt) {
                c[i] = add2(dr[i].wide(), u);
                u = fma2(nz[i], c[i], c[i]);
            }
#pragma unroll
        for (int i = 0; i < TS; ++i)
            if (i < cnt) {
                const float2 xi = xr[i].wide();
                ln.store(dx + (long long)(t0 + i) * prm.dx.st, mul2(neg2(nz[i]), c[i]));
                ln.store(dg + (long long)(t0 + i) * prm.dg.st, mul2(mul2(za[i], c[i]), add2(h, neg2(xi))));
                h = fma2(nz[i], neg2(xi), fma2(nz[i], h, h));
            }
    }
    if (prm.dh0 != nullptr && warp == 0 && rank == 0) ln.store_state(prm.dh0 + (long long)n * prm.D, carry);
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
