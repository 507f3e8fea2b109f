// The gated recurrence, forward, backward and one token:
//
//   z_t = sigmoid(-g_t),  a_t = 1 - z_t = sigmoid(g_t);   h_t = a_t h_{t-1} + z_t x_t,   h_{-1} = the state a sequence starts from
//   c_t = dh_t + u_{t+1},  u_t = a_t c_t,  u after the last step = the gradient of the state it leaves;
//   dx_t = z_t c_t,   dg_t = c_t (h_{t-1} - x_t) z_t a_t,   gradient of the starting state = u_0
//
// Every channel of every sequence is a chain of its own, and over a stretch of steps both recurrences are affine maps with the
// same slope A = prod a_t: h -> A h + F and u -> A u + R. A step is taken as h - z h + z x with two fused operations: what is
// rounded is then small beside 1 - a where a gate holds the state for thousands of steps, which a = 1 - z rounded is not. Where a gate
// forgets it is taken as (x - a x) + a h (kForgetGate), and where a value is infinite as kCareInfinite says.
//
// A CTA owns 64 channels of one sequence and walks it in tiles of W x TS steps. Each warp takes TS consecutive steps
// of the tile, each lane two channels. The warp's rows come in by asynchronous copies into a ring of its own in shared memory,
// tiles ahead, so that what is in flight (64 KB an SM and more) does not hang on registers or on other warps; it composes the map
// of its steps, puts it in shared memory, and after one barrier folds the maps of the warps in front of it to get its own first
// state; then it walks its steps once more and stores. So every input is read and every output written once. The backward needs
// the states in front of its steps: the forward leaves one per kGatedUnit steps and channel, and the backward, whose tile is one
// such unit, walks forward from it in registers, which is 4 bytes per 64 steps to read in place of h.
// With a cluster of CTAs a sequence's tiles go round robin to its CTAs, which exchange their tiles' maps through distributed
// shared memory once a round: the way to fill the GPU with few sequences or channels.
//
// What bounds it: memory as long as the exponential and the two passes over a step's maps keep up. Forward a pair of steps costs 35
// instructions of a warp, backward 74, with half of the schedulers' slots used (a chain of 4 to 8 warps a scheduler). Measured in
// bfloat16: 4 x 8192 x 2048 forward 84 us (4.8 TB/s of x, g and h, of 6.55 that a copy reaches); 16 x 2048 x 1536 forward 59 us,
// backward 95 (5.3 TB/s); 1 x 65536 x 4096 forward 320 us (5.0 TB/s), backward 566 (4.7); float32, 16 x 2048 x 1536, forward 111 (5.4 TB/s),
// backward 171 (5.9). Not kept, as they were slower: eight steps a warp with three or four CTAs an SM, two chains a warp, z kept in
// shared memory, rings of more tiles.
#pragma once

#include <type_traits>

#include "kla_common.cuh"

namespace kla {

constexpr int kGatedChannels = 64;  // of a CTA
constexpr int kGatedUnit = 64;      // steps between the states the forward leaves for the backward
constexpr int kGatedMaxCluster = 8;
constexpr int kGatedSite = 0x50;  // of the status word: the wait for the other CTAs' maps

struct GatedParams {
    int N, L, D;        // sequences, rows of a batch entry (packed: of all sequences), channels
    int blocks;         // channel blocks
    int clears;         // of packed sequences
    Tensor3 x, g, h;
    int x_width, g_width, dh_width;  // bytes a copy of their rows may move (gated_fetch)
    const int *cu;      // [N + 1] bounds of packed sequences or nullptr: sequences are batch entries
    const float *h0;    // [N, D] or nullptr: zeros
    float *end;         // [N, D]
    float *ckpt;        // states the backward starts from, or nullptr
    Tensor3 dh, dx, dg;
    const float *dend;  // [N, D] or nullptr: zeros
    float *dh0;         // [N, D] or nullptr
    WaitCtl wait;
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
    __device__ __forceinline__ void put(float *row, float2 y) const {
        if constexpr (PAIR) {
            *reinterpret_cast<float2 *>(row + 2 * lane) = y;
        } else {
            row[lane] = y.x;
            row[lane + 32] = y.y;
        }
    }
    // -y to a row; `row` points at c0
    __device__ __forceinline__ void store_negated(float *row, float2 y) const {
        y = neg2(y);
        if constexpr (PAIR) {
            if (on0) *reinterpret_cast<float2 *>(row) = y;
        } else {
            if (on0) row[0] = y.x;
            if (on1) row[32] = y.y;
        }
    }
    __device__ __forceinline__ void store_negated(__nv_bfloat16 *row, float2 y) const {
        const __nv_bfloat162 v = __floats2bfloat162_rn(y.x, y.y);
        const uint32_t w = *reinterpret_cast<const uint32_t *>(&v) ^ 0x80008000u;  // one operation for both signs
        if constexpr (PAIR) {
            if (on0) *reinterpret_cast<uint32_t *>(row) = w;
        } else {
            if (on0) reinterpret_cast<unsigned short *>(row)[0] = (unsigned short)w;
            if (on1) reinterpret_cast<unsigned short *>(row)[32] = (unsigned short)(w >> 16);
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
// the tensor's are zeros, rows past the sequence's `fill`. src: at the block's first channel. Any tile; gated_fetch has its own way
// for whole tiles of aligned rows.
template <typename T, int TS>
__device__ __noinline__ void gated_fetch_any(T *dst, const T *src, long long stride, int rows, int channels, int width, int lane, float fill) {
    if (rows < TS)
        for (int i = max(rows, 0) * kGatedChannels + lane; i < TS * kGatedChannels; i += 32) dst[i] = from_f32<T>(fill);
    if (width >= 4) {
        const int per = width / (int)sizeof(T), pieces = kGatedChannels / per;
#pragma unroll 4
        for (int i = lane; i < rows * pieces && i < TS * pieces; i += 32) {
            const int r = i / pieces, c = (i - r * pieces) * per;
            const int bytes = max(0, min(width, (channels - c) * (int)sizeof(T)));  // (pairs of bfloat16: channels is even)
            gated_copy(dst + r * kGatedChannels + c, bytes > 0 ? src + r * stride + c : src, bytes, width == 16);
        }
    } else {
        const int n0 = lane < channels, n1 = lane + 32 < channels;
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
// A warp's tiles of one tensor: src moves on from tile to tile.
template <typename T, int TS>
struct GatedRows {
    static constexpr int kPer = 16 / (int)sizeof(T), kPieces = kGatedChannels / kPer, kRows = 32 / kPieces;  // rows a warp's copies of 16 bytes cover
    const T *src;         // the next tile's first row, at the block's first channel
    long long stride, tile;  // elements between rows, to the next tile
    int channels, width, lane, bytes;
    float fill;
    __device__ __forceinline__ GatedRows(const T *rows, long long stride_, long long t0, long long tile_rows, int block, int D, int width_, int lane_, float fill_)
        : src(rows + t0 * stride_ + block * kGatedChannels), stride(stride_), tile(tile_rows * stride_), channels(D - block * kGatedChannels), width(width_),
          lane(lane_), fill(fill_) {
        bytes = max(0, min(16, (channels - lane % kPieces * kPer) * (int)sizeof(T)));
    }
    __device__ __forceinline__ void fetch(T *dst, int rows) {
        if (width == 16 && rows >= TS) {
            const T *from = src + lane / kPieces * stride + (bytes > 0 ? lane % kPieces * kPer : 0);
            T *to = dst + lane / kPieces * kGatedChannels + lane % kPieces * kPer;
            const long long next = kRows * stride;
#pragma unroll
            for (int i = 0; i < TS; i += kRows) {
                gated_copy(to + i * kGatedChannels, from, bytes, true);
                from += next;
            }
        } else if (width == 4 && rows >= TS) {
            constexpr int kWord = 4 / (int)sizeof(T);
#pragma unroll
            for (int h = 0; h < kGatedChannels / kWord / 32; ++h) {
                const int c = (lane + 32 * h) * kWord, there = c < channels ? 4 : 0;  // (pairs of bfloat16: channels is even)
                const T *from = src + (there ? c : 0);
#pragma unroll
                for (int i = 0; i < TS; ++i) {
                    gated_copy(dst + i * kGatedChannels + c, from, there, false);
                    from += stride;
                }
            }
        } else {
            gated_fetch_any<T, TS>(dst, src, stride, rows, channels, width, lane, fill);
        }
        src += tile;
    }
};
__device__ __forceinline__ void gated_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void gated_arrived() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    __syncwarp();
}

// Warps of a CTA, steps of a warp in a tile, tiles of its ring, CTAs an SM holds.
template <typename T>
struct GatedFwdShape {
    static constexpr int W = 4, TS = 64 / (int)sizeof(T), S = 2, kCtas = 3;
    static constexpr size_t kBytes = (size_t)W * S * 2 * TS * kGatedChannels * sizeof(T);
};
template <typename T>
struct GatedBwdShape {
    static constexpr int W = 4, TS = kGatedUnit / W, S = 2, kCtas = sizeof(T) == 2 ? 3 : 2;
    static constexpr size_t kBytes = (size_t)W * S * 3 * TS * kGatedChannels * sizeof(T);
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

// Rows in front of the first and behind the last packed sequence belong to none: zeros, by `clears` cells of the grid a block. (Going
// through all rows to find these took longer than the scan: 40 sequences in 32768 rows of 1536, bfloat16,
// backward 382 us in place of 133.)
template <typename T, bool PAIR>
__device__ __forceinline__ void gated_clear(const GatedParams &p, const Tensor3 &t, const Lane<PAIR> &ln, int cell, int warp, int warps, int rank, int ranks) {
    const int first = min(max(p.cu[0], 0), p.L), last = min(max(p.cu[p.N], 0), p.L);
    const int r0 = (cell * ranks + rank) * warps + warp, step = p.clears * ranks * warps;
    T *to = static_cast<T *>(const_cast<void *>(t.ptr)) + ln.c0;
    for (int r = r0; r < first; r += step) ln.store_negated(to + (long long)r * t.st, make_float2(-0.0f, -0.0f));
    for (int r = last + r0; r < p.L; r += step) ln.store_negated(to + (long long)r * t.st, make_float2(-0.0f, -0.0f));
}

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHold = 1e30f;  // a gate that holds: z is exactly 0

// -z of gates: a gate of +-inf gives exactly 0 or -1
__device__ __forceinline__ float2 gate_nz(float2 g) {
    const float2 t = mul2(g, dup2(kLog2e)), d = fma2(make_float2(ex2_approx(t.x), ex2_approx(t.y)), dup2(-1.0f), dup2(-1.0f));
    return make_float2(rcp_approx(d.x), rcp_approx(d.y));
}
// -z and z a, both with the relative accuracy of the smaller of z and a, and that smaller one
__device__ __forceinline__ void gate_slope(float2 g, float2 &nz, float2 &za, float2 &small) {
    const float2 e = make_float2(ex2_approx(fabsf(g.x) * -kLog2e), ex2_approx(fabsf(g.y) * -kLog2e)), d = add2(e, dup2(1.0f));
    const float2 r = make_float2(rcp_approx(d.x), rcp_approx(d.y));
    small = mul2(e, r);
    nz = make_float2(g.x >= 0.0f ? -small.x : -r.x, g.y >= 0.0f ? -small.y : -r.y);
    za = mul2(small, r);
}
// Where a gate forgets, v - z v is all cancellation: off by 2^-24 of v and more, it has few digits of a v left, or none. So a gate
// below kForgetGate is taken by a itself, which has full relative accuracy, and a step as (x - a x) + a h. Its factor w is a, with a
// positive sign (+0 too), in place of -z, whose sign is negative (-0 too). Above it a is at least 0.0025 in float32 and 0.00034 in
// bfloat16, so that 2^-23 of z are at most 2^-14 and 2^-11 of a. The choice costs instructions, and a warp makes it only in tiles
// that have such a gate, in loops that are not unrolled and a second time over the steps: unrolled beside the others, they took
// the backward without any such gate from 91 to 117 us (16 x 2048 x 1536, bfloat16; 94 as it is). Gates from kForgetGate on get the
// same bits either way. Measured at that shape, gates of mean 2 / of mean 0 and deviation 1.5 / of mean -6, us: float32 forward 111 /
// 112 / 128, backward 171 / 195 / 318; bfloat16 59 / 59 / 124, 95 / 95 / 230. What infinite values need is a third way (kCareInfinite), for
// tiles whose map turned out NaN or whose first state is infinite: within the second it would cost as much again.
template <typename T>
constexpr float kForgetGate = sizeof(T) == 2 ? -8.0f : -6.0f;
__device__ __forceinline__ bool forgets(float w) { return __float_as_int(w) >= 0; }
template <typename T>
__device__ __forceinline__ float2 chosen_factor(float2 g, float2 a, float2 nz) { return make_float2(g.x < kForgetGate<T> ? a.x : nz.x, g.y < kForgetGate<T> ? a.y : nz.y); }
// of the forward (its -z are gate_nz's)
template <typename T>
__device__ __forceinline__ float2 gate_factor(float2 g) {
    const float2 t = mul2(g, dup2(kLog2e)), e = make_float2(ex2_approx(t.x), ex2_approx(t.y)), d = fma2(e, dup2(-1.0f), dup2(-1.0f));
    const float2 nz = make_float2(rcp_approx(d.x), rcp_approx(d.y));
    return chosen_factor<T>(g, neg2(mul2(e, nz)), nz);
}
__device__ __forceinline__ float lowest(float low, float2 g) { return fminf(low, fminf(g.x, g.y)); }
// A step for two channels of the negated state, -h_t = -h + z h - z x, and the factor alone. (The state is carried negated because -z
// comes out of the gate and x out of memory as they are: each negation would be an operation a step.)
enum GatedCare {
    kCareNone = 0,      // no gate below kForgetGate
    kCareForgets = 1,
    kCareInfinite = 2   // also infinite values as the formula takes them: a inf is inf as long as a is not 0, where inf - z inf is NaN
};
__device__ __forceinline__ bool infinite(float v) { return fabsf(v) == __int_as_float(0x7f800000); }
__device__ __forceinline__ bool infinite(float2 v) { return infinite(v.x) || infinite(v.y); }
__device__ __forceinline__ bool nan(float2 v) { return v.x != v.x || v.y != v.y; }
template <int CARE>
__device__ __forceinline__ float2 factor_of(float2 v) {  // what a factor multiplies beside v itself
    return CARE == kCareInfinite ? make_float2(infinite(v.x) ? 0.0f : v.x, infinite(v.y) ? 0.0f : v.y) : v;
}
template <int CARE>
__device__ __forceinline__ float2 decay(float2 w, float2 v) {
    if (CARE == kCareNone) return fma2(w, v, v);
    const bool f0 = forgets(w.x), f1 = forgets(w.y);
    const float2 u = factor_of<CARE>(v);
    return fma2(w, make_float2(f0 ? v.x : u.x, f1 ? v.y : u.y), make_float2(f0 ? 0.0f : v.x, f1 ? 0.0f : v.y));
}
template <int CARE>
__device__ __forceinline__ float2 gate_step(float2 w, float2 x, float2 nh) {
    if (CARE == kCareNone) return fma2(w, x, fma2(w, nh, nh));
    // the larger term first: it alone cannot overflow
    const bool f0 = forgets(w.x), f1 = forgets(w.y);
    const float2 near = fma2(w, factor_of<CARE>(make_float2(f0 ? x.x : nh.x, f1 ? x.y : nh.y)), make_float2(f0 ? -x.x : nh.x, f1 ? -x.y : nh.y));
    return fma2(w, make_float2(f0 ? nh.x : x.x, f1 ? nh.y : x.y), near);
}

// A slope that fell below float32's range is its least number, not 0: an infinite state goes through it, as it does step by step.
// Only a factor of 0, a gate that leaves nothing, makes 0 (and NaN of an infinite state).
constexpr float kLeastSlope = 1.401298464e-45f;
__device__ __forceinline__ bool resets(float w) { return __float_as_uint(w) == 0u; }
__device__ __forceinline__ float slope_product(float a, float b) { return fmaxf(a * b, fminf(fminf(a, b), kLeastSlope)); }

// h -> A h + F of a stretch, two channels
struct Map2 {
    float2 A, F;
    __device__ __forceinline__ float2 operator()(float2 h) const { return make_float2(fmaf(A.x, h.x, F.x), fmaf(A.y, h.y, F.y)); }
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
__device__ __forceinline__ uint32_t at_rank(uint32_t here, uint32_t rank) {  // the address `here` has in another CTA of the cluster
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(rank));
    return there;
}
// 16 bytes into another CTA's shared memory, counted by a barrier of that CTA
__device__ __forceinline__ void cluster_send(uint32_t there, float4 v, uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(there), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(bar)
                 : "memory");
}

// Maps of the CTA's warps and (CLUSTER) of the cluster's CTAs, twice: a round writes one copy while the slowest reader of the
// round before may still be in the other.
// The CTAs' maps, [2][ranks][32] of 16 bytes, lie behind the ring: as many as there are, so that three CTAs of a cluster of up to six
// fit an SM.
constexpr size_t kGatedCtaMap = 2 * 32 * sizeof(float4);
template <bool CLUSTER, int W>
struct GatedShared {
    float4 warp[2][W][32];
    float2 carry[2][32];
    uint64_t arrived[2];  // (CLUSTER) of the copies: all CTAs' maps are here
};

// mbar_wait without sleeps between its polls (which suspend the thread themselves), counted in cycles of at most 2 GHz.
__device__ __forceinline__ bool gated_wait(const WaitCtl &w, uint64_t *bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long begin = clock64(), limit = 2ll * w.limit_ns;
    do {
        for (int i = 0; i < 32; ++i)
            if (mbar_try_wait(bar, parity)) return true;
    } while (clock64() - begin < limit);
    atomicCAS(w.status, 0, kStatusWait | kGatedSite);
    return false;
}

// Called by all threads with the map of the warp's own steps: the value in front of the warp's steps. The value in front of the round is
// sh.carry[buf] (for the first round put there by the warp that is last in the fold), the one behind it goes to the other copy.
// REVERSE: values come from behind. One barrier of the CTA. With CLUSTER the CTAs send one another their maps and wait for those of the
// others by a barrier that counts bytes: a barrier of the cluster would wait for every warp's stores to memory each round. A copy
// is written again two rounds later, by a CTA that has this CTA's map of the round between, which is sent behind the barrier that
// the copy's last reader has passed. ok: false once a bounded wait has run out; the thread then waits no more, but goes on with
// whatever is there, so that all threads meet in the remaining barriers and the kernel ends.
template <bool CLUSTER, bool REVERSE, int W>
__device__ __forceinline__ float2 gated_exchange(GatedShared<CLUSTER, W> &sh, float4 *ctas, const WaitCtl &wait, int round, Map2 own, int warp, int lane, int rank, int ranks, bool &ok) {
    const int buf = round & 1;
    ctas += buf * ranks * 32 + lane;  // of this copy
    auto map = [](const float4 &v) { return Map2{make_float2(v.x, v.y), make_float2(v.z, v.w)}; };
    const int place = REVERSE ? W - 1 - warp : warp;  // in the order of the fold
    sh.warp[buf][place][lane] = make_float4(own.A.x, own.A.y, own.F.x, own.F.y);
    __syncthreads();
    float2 mine;
    if constexpr (CLUSTER) {
        if (warp == 0) {  // the CTA's map to all
            Map2 all{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const Map2 m = map(sh.warp[buf][i][lane]);
                all.F = m(all.F);
                all.A = make_float2(slope_product(m.A.x, all.A.x), slope_product(m.A.y, all.A.y));
            }
            const float4 v = make_float4(all.A.x, all.A.y, all.F.x, all.F.y);
            const uint32_t here = smem_u32(ctas + rank * 32), bar = smem_u32(&sh.arrived[buf]);
            // (not after a wait that ran out: its barrier's phase is not complete, and a second arrival in one phase is an error)
            if (ok && lane == 0) mbar_arrive_expect_tx(&sh.arrived[buf], ranks * 512);
            if (ok && round != wait.skip_tile)  // skip_tile: the tests' incomplete hand-over
                for (int r = 0; r < ranks; ++r) cluster_send(at_rank(here, r), v, at_rank(bar, r));
        }
        ok = ok && gated_wait(wait, &sh.arrived[buf], (round >> 1) & 1);
        mine = sh.carry[buf][lane];
        const int before = REVERSE ? ranks - 1 - rank : rank;
        for (int i = 0; i < before; ++i) mine = map(ctas[(REVERSE ? ranks - 1 - i : i) * 32])(mine);
        if (place == W - 1) {  // (the warp that folds most anyway)
            float2 end = mine;
            for (int i = before; i < ranks; ++i) end = map(ctas[(REVERSE ? ranks - 1 - i : i) * 32])(end);
            sh.carry[buf ^ 1][lane] = end;
        }
    } else {
        mine = sh.carry[buf][lane];
    }
#pragma unroll
    for (int i = 0; i < W - 1; ++i)
        if (i < place) mine = map(sh.warp[buf][i][lane])(mine);
    if (!CLUSTER && place == W - 1) sh.carry[buf ^ 1][lane] = own(mine);
    return mine;
}

// Grid: sequences x channel blocks x cluster, the last fastest; behind packed sequences `clears` more, which clear the rows that
// belong to none.
template <typename T, bool PAIR, bool CLUSTER>
__global__ void __launch_bounds__(GatedFwdShape<T>::W * 32, GatedFwdShape<T>::kCtas) kla_gated_fwd_kernel(const __grid_constant__ GatedParams prm) {
    using Shape = GatedFwdShape<T>;
    constexpr int W = Shape::W, TS = Shape::TS, S = Shape::S, TT = W * TS;
    __shared__ GatedShared<CLUSTER, W> sh;
    extern __shared__ __align__(16) unsigned char ring_bytes[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = CLUSTER ? (int)cluster_rank() : 0, ranks = CLUSTER ? (int)cluster_size() : 1;
    const int cell = blockIdx.x / ranks, n = cell / prm.blocks, block = cell % prm.blocks;
    const Lane<PAIR> ln(block, lane, prm.D);
    if (n >= prm.N) return gated_clear<T, PAIR>(prm, prm.h, ln, n - prm.N, warp, W, rank, ranks);  // the whole cluster returns
    if constexpr (CLUSTER) {
        if (threadIdx.x == 0) {
            mbar_init(&sh.arrived[0], 1);
            mbar_init(&sh.arrived[1], 1);
            mbar_fence_init();
        }
        cluster_sync();  // every CTA has begun: its shared memory may be written
    }
    bool ok = true;
    const GatedSpan span = gated_span(prm, n);
    const T *x = gated_rows<const T>(prm.x, span), *g = gated_rows<const T>(prm.g, span);
    T *h_out = gated_rows<T>(prm.h, span);
    T *ring = reinterpret_cast<T *>(ring_bytes) + warp * S * 2 * TS * kGatedChannels;
    float4 *ctas = reinterpret_cast<float4 *>(ring_bytes + Shape::kBytes);
    const int rounds = (span.len + TT * ranks - 1) / (TT * ranks), len = span.len;
    if (warp == W - 1) sh.carry[0][lane] = prm.h0 ? neg2(ln.load_state(prm.h0 + (long long)n * prm.D)) : make_float2(0.0f, 0.0f);

    const int first = rank * TT + warp * TS;
    GatedRows<T, TS> gates(g, prm.g.st, first, (long long)ranks * TT, block, prm.D, prm.g_width, lane, kHold);
    GatedRows<T, TS> inputs(x, prm.x.st, first, (long long)ranks * TT, block, prm.D, prm.x_width, lane, 0.0f);
    int fetched = 0, slot_in = 0;
    auto fetch = [&] {  // the next round's rows, where there is one; a group of copies either way
        if (fetched < rounds) {
            const int rows = len - (fetched * ranks * TT + first);
            T *to = ring + slot_in * 2 * TS * kGatedChannels;
            gates.fetch(to, rows);
            inputs.fetch(to + TS * kGatedChannels, rows);
        }
        gated_commit();
        ++fetched;
        if (++slot_in == S) slot_in = 0;
    };
    int slot = 0;
    for (int round = 1 - S; round < rounds; ++round) {  // (the first S - 1 only fetch: one copy of that code)
        const int t0 = (round * ranks + rank) * TT + warp * TS, cnt = len - t0;
        if (round >= 0) gated_arrived<S - 2>();
        fetch();  // over the round before
        if (round < 0) continue;
        T *gs = ring + slot * 2 * TS * kGatedChannels, *xs = gs + TS * kGatedChannels;
        if (++slot == S) slot = 0;
        float2 nz[TS];
        Map2 own{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
        float low = 0.0f;
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            const float2 gate = ln.take(gs + i * kGatedChannels);
            low = lowest(low, gate);
            nz[i] = gate_nz(gate);
            own.A = decay<kCareNone>(nz[i], own.A);
            own.F = gate_step<kCareNone>(nz[i], ln.take(xs + i * kGatedChannels), own.F);
        }
        // The map with care, and the least its slope may be. float32 factors take the gates' place in shared memory, bfloat16 has no room for
        // them there and keeps them in local memory (which in float32 took 149 us in place of 127 at 16 x 2048 x 1536).
        float2 local[sizeof(T) == 2 ? TS : 1];
        bool made = false;
        auto factor = [&](int i) {
            if constexpr (sizeof(T) == 4) return ln.take(gs + i * kGatedChannels);
            else return local[i];
        };
        auto careful = [&](auto care_) {
            constexpr int CARE = decltype(care_)::value;
            own = Map2{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
            bool r0 = false, r1 = false;
#pragma unroll 4
            for (int i = 0; i < TS; ++i) {
                const float2 w = made ? factor(i) : gate_factor<T>(ln.take(gs + i * kGatedChannels));
                if constexpr (sizeof(T) == 4) ln.put(gs + i * kGatedChannels, w);
                else local[i] = w;
                r0 |= resets(w.x);
                r1 |= resets(w.y);
                own.A = decay<CARE>(w, own.A);
                own.F = gate_step<CARE>(w, ln.take(xs + i * kGatedChannels), own.F);
            }
            made = true;
            return make_float2(r0 ? 0.0f : kLeastSlope, r1 ? 0.0f : kLeastSlope);
        };
        float2 least = dup2(kLeastSlope);
        int care = kCareNone;
        if (__any_sync(0xffffffffu, low < kForgetGate<T> || nan(own.F))) {
            care = kCareForgets;
            least = careful(std::integral_constant<int, kCareForgets>{});
            if (__any_sync(0xffffffffu, nan(own.F))) {  // of an infinite value, or of the inputs
                care = kCareInfinite;
                careful(std::integral_constant<int, kCareInfinite>{});
            }
        }
        own.A = make_float2(fmaxf(own.A.x, least.x), fmaxf(own.A.y, least.y));
        float2 h = gated_exchange<CLUSTER, false, W>(sh, ctas, prm.wait, round, own, warp, lane, rank, ranks, ok);
        if (prm.ckpt != nullptr && t0 % kGatedUnit == 0 && cnt > 0)
            ln.store_state(prm.ckpt + (long long)(span.unit + t0 / kGatedUnit) * prm.D, neg2(h));
        if (__any_sync(0xffffffffu, infinite(h))) {
            care = kCareInfinite;
            if (!made) careful(std::integral_constant<int, kCareInfinite>{});
        }
        T *to = h_out + (long long)t0 * prm.h.st + ln.c0;
        auto walk = [&](auto care_) {
#pragma unroll 4
            for (int i = 0; i < min(cnt, TS); ++i) {
                h = gate_step<decltype(care_)::value>(factor(i), ln.take(xs + i * kGatedChannels), h);
                ln.store_negated(to, h);
                to += prm.h.st;
            }
        };
        if (care == kCareInfinite) {
            walk(std::integral_constant<int, kCareInfinite>{});
        } else if (care == kCareForgets) {
            walk(std::integral_constant<int, kCareForgets>{});
        } else if (cnt >= TS) {
#pragma unroll
            for (int i = 0; i < TS; ++i) {
                h = gate_step<kCareNone>(nz[i], ln.take(xs + i * kGatedChannels), h);
                ln.store_negated(to, h);
                to += prm.h.st;
            }
        } else {
#pragma unroll
            for (int i = 0; i < TS; ++i)
                if (i < cnt) {
                    h = gate_step<kCareNone>(nz[i], ln.take(xs + i * kGatedChannels), h);
                    ln.store_negated(to, h);
                    to += prm.h.st;
                }
        }
    }
    if constexpr (CLUSTER) cluster_sync();  // no CTA leaves while another may send to it (all has arrived, unless a wait ran out)
    if (warp == W - 1 && rank == 0) ln.store_state(prm.end + (long long)n * prm.D, neg2(sh.carry[rounds & 1][lane]));  // its own
}

template <typename T, bool PAIR, bool CLUSTER>
__global__ void __launch_bounds__(GatedBwdShape<T>::W * 32, GatedBwdShape<T>::kCtas) kla_gated_bwd_kernel(const __grid_constant__ GatedParams prm) {
    using Shape = GatedBwdShape<T>;
    constexpr int W = Shape::W, TS = Shape::TS, S = Shape::S, kTile = TS * kGatedChannels;
    __shared__ GatedShared<CLUSTER, W> sh;
    __shared__ float4 fw[2][W][32];  // maps of the warps forwards
    extern __shared__ __align__(16) unsigned char ring_bytes[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = CLUSTER ? (int)cluster_rank() : 0, ranks = CLUSTER ? (int)cluster_size() : 1;
    const int cell = blockIdx.x / ranks, n = cell / prm.blocks, block = cell % prm.blocks;
    const Lane<PAIR> ln(block, lane, prm.D);
    if (n >= prm.N) {
        gated_clear<T, PAIR>(prm, prm.dx, ln, n - prm.N, warp, W, rank, ranks);
        return gated_clear<T, PAIR>(prm, prm.dg, ln, n - prm.N, warp, W, rank, ranks);
    }
    if constexpr (CLUSTER) {
        if (threadIdx.x == 0) {
            mbar_init(&sh.arrived[0], 1);
            mbar_init(&sh.arrived[1], 1);
            mbar_fence_init();
        }
        cluster_sync();
    }
    bool ok = true;
    const GatedSpan span = gated_span(prm, n);
    const T *x = gated_rows<const T>(prm.x, span), *g = gated_rows<const T>(prm.g, span), *dh = gated_rows<const T>(prm.dh, span);
    T *dx = gated_rows<T>(prm.dx, span), *dg = gated_rows<T>(prm.dg, span);
    T *ring = reinterpret_cast<T *>(ring_bytes) + warp * S * 3 * kTile;
    float4 *ctas = reinterpret_cast<float4 *>(ring_bytes + Shape::kBytes);
    const int len = span.len, rounds = (len + kGatedUnit * ranks - 1) / (kGatedUnit * ranks);
    // copies of the exchange by parity of the rounds done
    if (warp == 0) sh.carry[0][lane] = prm.dend ? ln.load_state(prm.dend + (long long)n * prm.D) : make_float2(0.0f, 0.0f);

    const int first = ((rounds - 1) * ranks + rank) * kGatedUnit + warp * TS;  // the last round's
    const long long tile = -(long long)ranks * kGatedUnit;
    GatedRows<T, TS> gates(g, prm.g.st, first, tile, block, prm.D, prm.g_width, lane, kHold);
    GatedRows<T, TS> inputs(x, prm.x.st, first, tile, block, prm.D, prm.x_width, lane, 0.0f);
    GatedRows<T, TS> grads(dh, prm.dh.st, first, tile, block, prm.D, prm.dh_width, lane, 0.0f);
    int fetched = rounds - 1, slot_in = 0;
    auto fetch = [&] {  // rounds from the last one on
        if (fetched >= 0) {
            const int rows = len - ((fetched * ranks + rank) * kGatedUnit + warp * TS);
            T *to = ring + slot_in * 3 * kTile;
            gates.fetch(to, rows);
            inputs.fetch(to + kTile, rows);
            grads.fetch(to + 2 * kTile, rows);
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
    float2 next = front(rounds - 1);
    int slot = 0;
    for (int round = rounds - 2 + S; round >= 0; --round) {  // (the first S - 1 only fetch)
        const int t0 = (round * ranks + rank) * kGatedUnit + warp * TS, cnt = len - t0, buf = (rounds - 1 - round) & 1;
        if (round < rounds) gated_arrived<S - 2>();
        fetch();
        if (round >= rounds) continue;
        float2 h = neg2(next);  // (here, not where it is loaded: that would wait for it)
        next = front(round - 1);
        T *gs = ring + slot * 3 * kTile, *xs = gs + kTile, *ds = xs + kTile;
        if (++slot == S) slot = 0;
        float2 nz[TS], za[TS], c[TS];
        Map2 back{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
        float2 F = make_float2(0.0f, 0.0f);
        float low = 0.0f;
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            const float2 gate = ln.take(gs + i * kGatedChannels);
            low = lowest(low, gate);
            float2 small;
            gate_slope(gate, nz[i], za[i], small);
            back.A = decay<kCareNone>(nz[i], back.A);
            F = gate_step<kCareNone>(nz[i], ln.take(xs + i * kGatedChannels), F);
        }
        auto behind = [&](int i, float2 u) {  // the gradient that reaches step i
            const float2 d = ln.take(ds + i * kGatedChannels);
            return add2(d, u);
        };
#pragma unroll
        for (int i = TS - 1; i >= 0; --i) back.F = decay<kCareNone>(nz[i], behind(i, back.F));
        // With care the factors go through local memory, and c, which in float32 takes the place of dh.
        float2 factors[TS], local_c[sizeof(T) == 2 ? TS : 1];
        auto slopes = [&](int i, float2 &n, float2 &s) {
            const float2 gate = ln.take(gs + i * kGatedChannels);
            float2 small;
            gate_slope(gate, n, s, small);
            return chosen_factor<T>(gate, small, n);
        };
        bool made = false;
        auto careful = [&](auto care_) {
            constexpr int CARE = decltype(care_)::value;
            back = Map2{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
            F = make_float2(0.0f, 0.0f);
            bool r0 = false, r1 = false;
#pragma unroll 4
            for (int i = 0; i < TS; ++i) {
                float2 n, s;
                const float2 w = slopes(i, n, s);
                factors[i] = w;
                r0 |= resets(w.x);
                r1 |= resets(w.y);
                back.A = decay<CARE>(w, back.A);
                F = gate_step<CARE>(w, ln.take(xs + i * kGatedChannels), F);
            }
#pragma unroll 4
            for (int i = TS - 1; i >= 0; --i) back.F = decay<CARE>(factors[i], behind(i, back.F));
            made = true;
            return make_float2(r0 ? 0.0f : kLeastSlope, r1 ? 0.0f : kLeastSlope);
        };
        float2 least = dup2(kLeastSlope);
        int care = kCareNone;
        if (__any_sync(0xffffffffu, low < kForgetGate<T> || nan(F) || nan(back.F))) {
            care = kCareForgets;
            least = careful(std::integral_constant<int, kCareForgets>{});
            if (__any_sync(0xffffffffu, nan(F) || nan(back.F))) {
                care = kCareInfinite;
                careful(std::integral_constant<int, kCareInfinite>{});
            }
        }
        back.A = make_float2(fmaxf(back.A.x, least.x), fmaxf(back.A.y, least.y));
        fw[buf][warp][lane] = make_float4(back.A.x, back.A.y, F.x, F.y);
        float2 u = gated_exchange<CLUSTER, true, W>(sh, ctas, prm.wait, rounds - 1 - round, back, warp, lane, rank, ranks, ok);
#pragma unroll
        for (int w = 0; w < W - 1; ++w)
            if (w < warp) {
                const float4 m = fw[buf][w][lane];
                h = Map2{make_float2(m.x, m.y), make_float2(m.z, m.w)}(h);
            }
        if (__any_sync(0xffffffffu, infinite(u) || infinite(h))) {
            care = kCareInfinite;
            if (!made) careful(std::integral_constant<int, kCareInfinite>{});
        }
        T *to_x = dx + (long long)t0 * prm.dx.st + ln.c0, *to_g = dg + (long long)t0 * prm.dg.st + ln.c0;
        auto walk = [&](auto care_) {
            constexpr int CARE = decltype(care_)::value;
#pragma unroll 4
            for (int i = TS - 1; i >= 0; --i) {
                const float2 ci = behind(i, u);
                if constexpr (sizeof(T) == 4) ln.put(ds + i * kGatedChannels, ci);
                else local_c[i] = ci;
                u = decay<CARE>(factors[i], ci);
            }
#pragma unroll 4
            for (int i = 0; i < min(cnt, TS); ++i) {
                float2 n, s, ci;
                if constexpr (sizeof(T) == 4) ci = ln.take(ds + i * kGatedChannels);
                else ci = local_c[i];
                const float2 xi = ln.take(xs + i * kGatedChannels), w = slopes(i, n, s);
                ln.store_negated(to_x, mul2(n, ci));
                ln.store_negated(to_g, mul2(mul2(s, ci), add2(h, xi)));
                to_x += prm.dx.st;
                to_g += prm.dg.st;
                h = gate_step<CARE>(w, xi, h);
            }
        };
        if (care != kCareNone) {
            if (care == kCareInfinite) walk(std::integral_constant<int, kCareInfinite>{});
            else walk(std::integral_constant<int, kCareForgets>{});
            continue;
        }
#pragma unroll
        for (int i = TS - 1; i >= 0; --i) {
            c[i] = behind(i, u);
            u = decay<kCareNone>(nz[i], c[i]);
        }
        auto out = [&](int i) {  // h: negated
            const float2 xi = ln.take(xs + i * kGatedChannels);
            ln.store_negated(to_x, mul2(nz[i], c[i]));
            ln.store_negated(to_g, mul2(mul2(za[i], c[i]), add2(h, xi)));
            to_x += prm.dx.st;
            to_g += prm.dg.st;
            h = gate_step<kCareNone>(nz[i], xi, h);
        };
        if (cnt >= TS) {
#pragma unroll
            for (int i = 0; i < TS; ++i) out(i);
        } else {
#pragma unroll
            for (int i = 0; i < TS; ++i)
                if (i < cnt) out(i);
        }
    }
    if constexpr (CLUSTER) cluster_sync();
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
    const float2 g = make_float2(to_f32<T>(static_cast<const T *>(prm.g)[b * prm.g_sb + d]), 0.0f);
    const float2 w = gate_factor<float>(g);
    const float h = -gate_step<kCareInfinite>(w, make_float2(x, 0.0f), make_float2(-prm.state[i], 0.0f)).x;
    prm.state_out[i] = h;
    static_cast<T *>(prm.h)[i] = from_f32<T>(h);
}

}  // namespace kla
