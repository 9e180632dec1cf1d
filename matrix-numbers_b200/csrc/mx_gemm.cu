// Products of microscaled (MX) operands on the 5th-generation tensor cores, plain and grouped by expert:
//   C[i][j] = sum_l A[i][l] B[j][l],   A[i][l] = a 2^(sa - 127), B[j][l] = b 2^(sb - 127), scales shared by 32 l's.
// tcgen05.mma multiplies the codes, applies both scales to each block's partial sum and accumulates in FP32 in TMEM, so
// nothing is unpacked on the way: kind::mxf4 for two 4-bit operands (K = 64 an instruction), kind::mxf8f6f4 otherwise
// (K = 32; a 4-bit operand is spread to one code a byte by its TMA load).
//
// One persistent kernel, one CTA per SM:
//   - warp 0: producer; a stage is 128 bytes of K of 128 "left" rows (M) and BN "right" rows (N) and their
//     scale tiles, four TMA loads, the codes with the 128-byte swizzle;
//   - warp 1: lays a stage's scales into TMEM (tcgen05.cp, two buffers of columns), a stage ahead of the four
//     MMAs that use them, and issues those;
//   - warps 2..9: epilogue, TMEM -> registers -> one rounding -> C.
// Left is A and right is B (`SWAP` false), or, for few rows of A, left is B and right is A: the 128 rows that the
// instruction has at least are then rows of B, which there are plenty of, and A's tile is as small as 32 rows; C^T comes
// out of TMEM, whose lanes are then neighbours in a row of C.
// `PAIR`: two CTAs on neighbouring SMs share a 256 x 256 tile (cta_group::2): each holds 128 left rows and 128 right rows,
// so a stage of the same work brings 32 KB of codes to an SM instead of 48 KB, which its shared memory would take 768 clocks
// to write and read at 128 bytes a clock; the MMAs need 512 (2048 x 4096 x 4096 in e4m3: 28.7 us against 37.6).
// Where there are fewer tiles than SMs, a cluster of CTAs shares one tile: each takes a part of K, leaves its FP32 sums
// in its shared memory, and every CTA adds one slice of the tile over the cluster in a fixed order (no workspace, no
// atomics, one launch).
// Grouped: `ends` is read on the device; a group's rows are covered by windows of A (of a tile's rows, from the multiple of
// 128 at or before the group's first), and each window is multiplied with the group's B and stored for the group's rows
// only.  So A's rows and scales stay where the quantisation put them, whatever the routing, for at
// most one more tile per group than packing would need.
// The producer and the issuing warp run their loops as whole warps and let one elected lane issue: with the loops in one
// lane alone each operand of a tcgen05 instruction was moved to a uniform register on its way, and the issue bound the
// kernel (8192 x 4096 x 8192 in e2m1: 163 us, tensor pipe 41 % active; elected: 102 us, 70 %).
// Measured on one B200 at its power cap (1.4 - 1.5 GHz): e2m1 16384 x 8192 x 8192 in 392 us, 5.6 PFLOP/s; e4m3 8192 x 8192 x
// 8192 in 394 - 414 us, 2.7 - 2.8 PFLOP/s: four and two times the rate that the card sustains in bf16, and bound by the same cap.
// Every mbarrier wait is bounded; when a role's wait runs out it records a flag in *err and raises the CTA's abort flag (both
// CTAs' of a pair), through which the other roles leave.  When all have, whichever it was, the CTA waits (bounded) for its
// loads and MMAs in flight, frees TMEM and exits.  No multicast is used.
#include <cuda.h>

#include <atomic>

#include "mx_common.cuh"
#include "tc_ptx.cuh"

using namespace ozk_mx;
using namespace ozk_ptx;

namespace {

constexpr int BM = 128;                      // rows of the left operand's tile
constexpr int ROW_BYTES = 128;               // K bytes of one stage row (shared memory)
constexpr int EPI_WARPS = 8;
constexpr uint32_t OUT_WARP_BYTES = 32 * 128;   // one epilogue warp's 32 rows of C, 128 bytes each
constexpr int THREADS = (2 + EPI_WARPS) * 32;
constexpr int GROUP_L = 16;                  // left tiles per raster group
constexpr uint64_t WAIT_LIMIT_NS = 4000000000ull;   // 4 s of wall time per wait
constexpr uint64_t DRAIN_LIMIT_NS = 1000000000ull;  // 1 s for each load, and for the MMAs, that were in flight at a timeout
constexpr int MXF4 = 0, MXF8F6F4 = 1;
constexpr size_t SMEM_MAX = 232448;
constexpr size_t TABLE_BYTES = (2 * (OZK_MX_MAX_GROUPS + 1) * 4 + 15) / 16 * 16;

template <int KIND, int BN, bool SWAP, bool PAIR>
struct Shape {
    static constexpr int CTAS = PAIR ? 2 : 1;
    static constexpr int BL = BM * CTAS;                        // left rows of a tile
    static constexpr int RN = BN / CTAS;                        // right rows that one CTA loads
    static constexpr int KT = KIND == MXF4 ? 2 : 1;             // scale tiles (128 elements of K) of a stage
    static constexpr int SUBS = (BN + TILE - 1) / TILE;         // row tiles of the right operand's scales
    static constexpr uint32_t L_BYTES = BM * ROW_BYTES, R_BYTES = RN * ROW_BYTES;
    static constexpr uint32_t SL_BYTES = KT * TILE_BYTES, SR_BYTES = SUBS * KT * TILE_BYTES;
    static constexpr uint32_t STAGE_BYTES = L_BYTES + R_BYTES + SL_BYTES + SR_BYTES;
    // where C leaves by TMA; not for B on the left (C^T), nor for groups of few rows (128 x 256 alone), whose rows seldom fill
    // a box: there the room is a fourth stage
    static constexpr bool BOXES = !SWAP && (PAIR || BN < 256);
    static constexpr uint32_t OUT_BYTES = BOXES ? EPI_WARPS * OUT_WARP_BYTES : 0;
    static constexpr int FIT = (int)((SMEM_MAX - 1024 - 256 - TABLE_BYTES - OUT_BYTES) / STAGE_BYTES);
    static constexpr int STAGES = FIT < 8 ? FIT : 8;
    static constexpr size_t SMEM = (size_t)STAGES * STAGE_BYTES + OUT_BYTES + 1024 + 256 + TABLE_BYTES;
    static constexpr int NUM_BARS = 2 * STAGES + 5;             // full[S], empty[S], acc_full[2], acc_empty[2], drain
    // TMEM: two accumulators, then two buffers of scale columns.  With BN = 256 the accumulators overlap by 48 columns,
    // which makes room for the scales: the epilogue reads the shared columns first, and the next tile waits for those.
    static constexpr int SCALE_COLS = KT * 4 * (1 + SUBS);
    static constexpr int ACC_STRIDE = BN == 256 ? 208 : BN;
    static constexpr int SCALE_BASE = ACC_STRIDE + BN;
    static constexpr int USED = SCALE_BASE + 2 * SCALE_COLS;
    static constexpr uint32_t TMEM_COLS = USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
    static constexpr int LAG = BN == 256 ? 1 : 2;               // tiles between an accumulator's drain and its next use
    static constexpr int HALF = BN / 2;                         // accumulator columns of one epilogue warp
    static constexpr int CHUNK = HALF < 32 ? HALF : 32;
    static_assert(USED <= 512 && NUM_BARS * 8 + 16 <= 256 && STAGES >= 3, "fits");
    static_assert(PAIR || (size_t)(BN + 4) * BM * 4 <= (size_t)STAGES * STAGE_BYTES, "a tile of partial sums fits into the stages");
    static_assert(!PAIR || BN == 256, "a pair's tile is 256 x 256");
};

struct Args {
    int l_rows, r_rows;                      // rows (per group) of the left and right operand
    int ktiles;                              // scale tiles along K
    int kblocks;                             // stages along K
    uint32_t load_bytes;                     // what the loads of a stage count on its barrier
    int groups;                              // 0: no groups
    const int32_t* ends;
    int tokens, n;                           // rows and columns of C
    int fill;
    void* C;
    long long ldc;
    int dtype;
    bool vec;                                // rows of C are 16-byte aligned, and tmC describes it
    uint32_t idesc;
    int32_t* err;
    uint64_t limit_ns;                       // of every wait of the roles
};

struct Unit {
    int rg;                                  // group of the right operand
    int l0, r0;                              // first left and right row of the tile
    int first, last;                         // rows of A (and C) that belong to this unit's group: [first, last)
};

template <int BL, int BN>
struct Work {
    const Args& a;
    const int *pre, *bound;                  // grouped: windows before group g, first row of group g
    int ltiles, rtiles;
    long long units;

    __device__ Work(const Args& a_, const int* pre_, const int* bound_) : a(a_), pre(pre_), bound(bound_) {
        ltiles = (a.l_rows + BL - 1) / BL;
        rtiles = (a.r_rows + BN - 1) / BN;
        units = (long long)(a.groups ? pre[a.groups] : ltiles) * rtiles;
    }
    __device__ __forceinline__ Unit at(long long u) const {
        Unit w;
        if (a.groups) {                      // A is on the left; a group's windows next to each other, for B's columns in L2
            const int q = (int)(u / rtiles);
            int lo = 0, hi = a.groups - 1;                  // the last group with pre[g] <= q: it has windows
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (pre[mid] <= q) lo = mid; else hi = mid - 1;
            }
            w.first = bound[lo];
            w.last = bound[lo + 1];
            const long long in = u - (long long)pre[lo] * rtiles;
            const int nw = pre[lo + 1] - pre[lo];
            w.l0 = w.first / TILE * TILE + (int)(in % nw) * BL;
            w.r0 = (int)(in / nw) * BN;
            w.rg = lo;
        } else {
            const int per = GROUP_L * rtiles;
            const int g = (int)(u / per), l0 = g * GROUP_L, gl = min(ltiles - l0, GROUP_L);
            const int in = (int)(u - (long long)g * per);
            w.l0 = (l0 + in % gl) * BL;
            w.r0 = in / gl * BN;
            w.rg = 0;
            w.first = 0;
            w.last = a.tokens;
        }
        return w;
    }
};

__device__ __forceinline__ uint32_t pack2(float a, float b, int dtype) {
    if (dtype == OZK_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void store1(void* C, long long at, float v, int dtype) {
    if (dtype == OZK_F32) static_cast<float*>(C)[at] = v;
    else if (dtype == OZK_BF16) static_cast<__nv_bfloat16*>(C)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(C)[at] = __float2half_rn(v);
}

// Four words of 32 bytes that a pair of lanes holds for two rows of C: the even lane's row gets both lanes' low or high
// half in one store, then the odd lane's, so that every store of the warp fills whole 32-byte sectors.
__device__ __forceinline__ void store_pair(uint8_t* even_row, uint8_t* odd_row, bool even_in, bool odd_in, bool odd_lane,
                                           const uint32_t (&w)[8]) {
    uint4 own, got;
    own.x = odd_lane ? w[4] : w[0]; own.y = odd_lane ? w[5] : w[1]; own.z = odd_lane ? w[6] : w[2]; own.w = odd_lane ? w[7] : w[3];
    got.x = __shfl_xor_sync(0xffffffffu, odd_lane ? w[0] : w[4], 1);
    got.y = __shfl_xor_sync(0xffffffffu, odd_lane ? w[1] : w[5], 1);
    got.z = __shfl_xor_sync(0xffffffffu, odd_lane ? w[2] : w[6], 1);
    got.w = __shfl_xor_sync(0xffffffffu, odd_lane ? w[3] : w[7], 1);
    const int at = odd_lane ? 16 : 0;
    if (even_in) *reinterpret_cast<uint4*>(even_row + at) = odd_lane ? got : own;
    if (odd_in) *reinterpret_cast<uint4*>(odd_row + at) = odd_lane ? own : got;
}

// One thread's CHUNK consecutive accumulator columns (`r` the first one's right row, `l` the lane's left row) to C; called
// by whole warps
template <int CHUNK, bool SWAP>
__device__ __forceinline__ void store_chunk(const Args& a, const Unit& w, int l, int r, const uint32_t (&v)[CHUNK]) {
    if (SWAP) {                              // l: column of C, r: row of C; the warp's lanes are neighbours in a row
        if (l >= a.n) return;
#pragma unroll
        for (int e = 0; e < CHUNK; e++)
            if (r + e >= w.first && r + e < w.last)
                store1(a.C, (long long)(r + e) * a.ldc + l, __uint_as_float(v[e]), a.dtype);
        return;
    }
    if (r >= a.n) return;
    if (a.vec && r + CHUNK <= a.n) {
        const int le = l & ~1, lo = l | 1, size = a.dtype == OZK_F32 ? 4 : 2;
        const bool even_in = le >= w.first && le < w.last, odd_in = lo >= w.first && lo < w.last, odd_lane = l & 1;
        uint8_t* pe = static_cast<uint8_t*>(a.C) + ((long long)le * a.ldc + r) * size;
        uint8_t* po = pe + a.ldc * size;
        if (a.dtype == OZK_F32) {
#pragma unroll
            for (int q = 0; q < CHUNK / 8; q++) {
                uint32_t p[8];
#pragma unroll
                for (int j = 0; j < 8; j++) p[j] = v[8 * q + j];
                store_pair(pe + 32 * q, po + 32 * q, even_in, odd_in, odd_lane, p);
            }
        } else {
#pragma unroll
            for (int q = 0; q < CHUNK / 16; q++) {
                uint32_t p[8];
#pragma unroll
                for (int j = 0; j < 8; j++)
                    p[j] = pack2(__uint_as_float(v[16 * q + 2 * j]), __uint_as_float(v[16 * q + 2 * j + 1]), a.dtype);
                store_pair(pe + 32 * q, po + 32 * q, even_in, odd_in, odd_lane, p);
            }
        }
    } else if (l >= w.first && l < w.last) {
        const long long at = (long long)l * a.ldc + r;
#pragma unroll
        for (int e = 0; e < CHUNK; e++)
            if (r + e < a.n) store1(a.C, at + e, __uint_as_float(v[e]), a.dtype);
    }
}

// One warp's 32 rows x 64 columns of the accumulator (rows from l0, columns from r) to C.  Whole row segments go through
// this warp's shared memory (128-byte swizzle) and leave by TMA, which clips at C's ends: 4.2 us an epilogue of 128 x 256
// with direct stores of 32 bytes a row, which were slower than the MMAs of K < 4096.  The edge rows of a group, and a C
// whose rows are not aligned, take the direct stores; so do the last columns where a row of C does not end on 16 bytes (a
// clipped box writes zeros up to there).
template <bool BOXES>
__device__ __forceinline__ void store_block(const Args& a, const CUtensorMap* tmC, const Unit& w, int l0, int r, int lane,
                                            uint32_t out, const uint32_t (&v0)[32], const uint32_t (&v1)[32]) {
    if (r >= a.n || l0 >= w.last || l0 + 32 <= w.first) return;
    const bool ends_inside = r + 64 > a.n && a.n * (a.dtype == OZK_F32 ? 4 : 2) % 16 != 0;
    if (!BOXES || !a.vec || ends_inside || l0 < w.first || (l0 + 32 > w.last && w.last < a.tokens)) {
        store_chunk<32, false>(a, w, l0 + lane, r, v0);
        store_chunk<32, false>(a, w, l0 + lane, r + 32, v1);
        return;
    }
    const uint32_t row = out + (uint32_t)lane * 128u, sw = (uint32_t)(lane & 7);
    auto ready = [&] {                          // the box that was here has been read
        if (lane == 0) bulk_wait_read();
        __syncwarp();
    };
    auto send = [&](int col) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(tmC, out, col, l0);
            bulk_commit();
        }
    };
    if (a.dtype == OZK_F32) {
        ready();
#pragma unroll
        for (int c = 0; c < 8; c++) st_shared_v4(row + (((uint32_t)c ^ sw) << 4), v0[4 * c], v0[4 * c + 1], v0[4 * c + 2], v0[4 * c + 3]);
        send(r);
        if (r + 32 >= a.n) return;
        ready();
#pragma unroll
        for (int c = 0; c < 8; c++) st_shared_v4(row + (((uint32_t)c ^ sw) << 4), v1[4 * c], v1[4 * c + 1], v1[4 * c + 2], v1[4 * c + 3]);
        send(r + 32);
    } else {
        uint32_t p[32];
#pragma unroll
        for (int j = 0; j < 16; j++) {
            p[j] = pack2(__uint_as_float(v0[2 * j]), __uint_as_float(v0[2 * j + 1]), a.dtype);
            p[16 + j] = pack2(__uint_as_float(v1[2 * j]), __uint_as_float(v1[2 * j + 1]), a.dtype);
        }
        ready();
#pragma unroll
        for (int c = 0; c < 8; c++) st_shared_v4(row + (((uint32_t)c ^ sw) << 4), p[4 * c], p[4 * c + 1], p[4 * c + 2], p[4 * c + 3]);
        send(r);
    }
}

// Four neighbouring values of a row of C
__device__ __forceinline__ void store4(const Args& a, int token, int col, float4 s) {
    const long long at = (long long)token * a.ldc + col;
    if (a.vec && col + 4 <= a.n) {
        if (a.dtype == OZK_F32) *reinterpret_cast<float4*>(static_cast<float*>(a.C) + at) = s;
        else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.C) + at) = make_uint2(pack2(s.x, s.y, a.dtype), pack2(s.z, s.w, a.dtype));
    } else {
        const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (col + e < a.n) store1(a.C, at + e, f[e], a.dtype);
    }
}

// Grouped: clamp `ends` to an ascending sequence within [0, rows] and count the windows each group touches (one warp)
template <int WIN>
__device__ __forceinline__ void group_tables(const Args& a, int* pre, int* bound, int lane) {
    int end_before = 0, windows_before = 0;
    if (lane == 0) { pre[0] = 0; bound[0] = 0; }
    for (int base = 0; base < a.groups; base += 32) {
        const int g = base + lane;
        int e = g < a.groups ? min(max(a.ends[g], 0), a.tokens) : 0;
        e = max(e, end_before);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int p = __shfl_up_sync(0xffffffffu, e, o);
            if (lane >= o) e = max(e, p);
        }
        int s = __shfl_up_sync(0xffffffffu, e, 1);
        if (lane == 0) s = end_before;
        int w = e > s ? (e - s / TILE * TILE + WIN - 1) / WIN : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int p = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += p;
        }
        w += windows_before;
        if (g < a.groups) { pre[g + 1] = w; bound[g + 1] = e; }
        end_before = __shfl_sync(0xffffffffu, e, 31);
        windows_before = __shfl_sync(0xffffffffu, w, 31);
    }
}

template <int CHUNK>
__device__ __forceinline__ void tmem_ld_chunk(uint32_t taddr, uint32_t (&v)[CHUNK]) {
    if constexpr (CHUNK == 32) tmem_ld_32x32b_x32(taddr, v);
    else tmem_ld_32x32b_x16(taddr, v);
}

template <int KIND, int BN, bool SWAP, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap tmL, const __grid_constant__ CUtensorMap tmR,
                   const __grid_constant__ CUtensorMap tmSL, const __grid_constant__ CUtensorMap tmSR,
                   const __grid_constant__ CUtensorMap tmC, const __grid_constant__ Args a, int parts) {
    using S = Shape<KIND, BN, SWAP, PAIR>;
    using WorkOf = Work<S::BL, BN>;
    constexpr int STAGES = S::STAGES, CHUNK = S::CHUNK;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sL = smem;
    uint8_t* sR = sL + STAGES * S::L_BYTES;
    uint8_t* sOut = sR + STAGES * S::R_BYTES;  // boxes of C on 1024-byte boundaries
    uint8_t* sSL = sOut + S::OUT_BYTES;
    uint8_t* sSR = sSL + STAGES * S::SL_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sSR + STAGES * S::SR_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::NUM_BARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile long long* peer_issued = reinterpret_cast<volatile long long*>(tmem_slot + 2);   // loads that CTA 1 of a pair issued
    int* pre = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + 256);
    int* bound = pre + OZK_MX_MAX_GROUPS + 1;

    // one value a warp, in a form that the compiler knows as such: the branches and loops that hang on it keep the operands
    // of the issuing warps in uniform registers
    auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const int warp = uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t bar0 = smem_addr(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * (uint32_t)s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (uint32_t)(STAGES + s); };
    auto accf_bar = [&](int b) { return bar0 + 8u * (uint32_t)(2 * STAGES + b); };
    auto acce_bar = [&](int b) { return bar0 + 8u * (uint32_t)(2 * STAGES + 2 + b); };
    const uint32_t drain_bar = bar0 + 8u * (uint32_t)(2 * STAGES + 4);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int b = 0; b < 2; b++) { mbar_init(accf_bar(b), 1); mbar_init(acce_bar(b), S::CTAS * EPI_WARPS); }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        if (PAIR) *peer_issued = 0;
        mbar_fence_init();
        tma_prefetch_desc(&tmL);
        tma_prefetch_desc(&tmR);
        tma_prefetch_desc(&tmSL);
        tma_prefetch_desc(&tmSR);
    }
    if (warp == 1) {
        if (PAIR) {
            tmem_alloc_pair(smem_addr(tmem_slot), S::TMEM_COLS);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_addr(tmem_slot), S::TMEM_COLS);
            tmem_relinquish();
        }
    }
    if (!SWAP && warp == 2 && a.groups) group_tables<S::BL>(a, pre, bound, lane);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();                  // the peer's barriers exist before any remote arrival
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    WorkOf work(a, pre, bound);
    work.units = (long long)(uint32_t)uniform((int)work.units) | (long long)uniform((int)(work.units >> 32)) << 32;
    // parts > 1: one unit per cluster of `parts` CTAs, each with its part of K; else units round robin over the CTAs, or
    // over the pairs, of which CTA 0 issues the MMAs
    const int rank = PAIR ? uniform((int)cluster_ctarank()) : 0;
    const int part = !PAIR && parts > 1 ? uniform((int)cluster_ctarank()) : 0;
    const long long u0 = blockIdx.x / (parts * S::CTAS), du = gridDim.x / (parts * S::CTAS);
    auto give_up = [&](int code) {             // one lane of a role whose wait ran out
        if (*abort_flag) return;               // it left through the flag: another role has reported
        *abort_flag = 1;
        if (PAIR) st_cluster_u32(map_to_rank(smem_addr(const_cast<const int*>(abort_flag)), (uint32_t)(rank ^ 1)), 1u);
        atomicOr(a.err, code);
    };
    auto commit = [&](uint32_t bar) {          // an arrival on that barrier of every CTA when all issued so far is done
        if (PAIR) {
            umma_commit_pair(map_to_rank(bar, 0u));
            umma_commit_pair(map_to_rank(bar, 1u));
        } else {
            umma_commit(bar);
        }
    };
    long long issued = 0;                      // loads, by the producer
    const int kb0 = (int)((long long)a.kblocks * part / parts), kb1 = (int)((long long)a.kblocks * (part + 1) / parts);

    if (warp == 0) {
        // ---------------------------------------------------------------- producer (the whole warp; one lane issues)
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        const uint32_t aL = smem_addr(sL), aR = smem_addr(sR), aSL = smem_addr(sSL), aSR = smem_addr(sSR);
        for (long long u = u0; ok && u < work.units; u += du) {
            const Unit w = work.at(u);
            const int l0 = uniform(w.l0) + rank * BM, rt = uniform(w.r0), r0 = rt + rank * S::RN;
            const int rg = uniform(w.rg);
            for (int kb = kb0; kb < kb1; kb++) {
                ok = mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, a.limit_ns);
                if (!ok) break;
                if (elect_one()) {
                    // a pair's loads all complete on CTA 0's barrier, which expects the bytes of both
                    if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), a.load_bytes * (uint32_t)S::CTAS);
                    const uint32_t bar = PAIR ? map_to_rank(full_bar(stage), 0u) : full_bar(stage);
                    const int kc = kb * (KIND == MXF4 ? ROW_BYTES : TILE);      // bytes (mxf4) or elements
                    const uint32_t dl = aL + stage * S::L_BYTES, dr = aR + stage * S::R_BYTES;
                    const uint32_t dsl = aSL + stage * S::SL_BYTES, dsr = aSR + stage * S::SR_BYTES;
                    if (PAIR) {
                        tma_load_3d_pair(dl, &tmL, kc, l0, 0, bar);
                        tma_load_3d_pair(dr, &tmR, kc, r0, rg, bar);
                        tma_load_4d_pair(dsl, &tmSL, 0, kb * S::KT, l0 / TILE, 0, bar);
                        tma_load_4d_pair(dsr, &tmSR, 0, kb * S::KT, rt / TILE, rg, bar);
                    } else {
                        tma_load_3d(dl, &tmL, kc, l0, 0, bar);
                        tma_load_3d(dr, &tmR, kc, r0, rg, bar);
                        tma_load_4d(dsl, &tmSL, 0, kb * S::KT, l0 / TILE, 0, bar);
                        tma_load_4d(dsr, &tmSR, 0, kb * S::KT, rt / TILE, rg, bar);
                    }
                }
                __syncwarp();
                issued++;
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
        }
        if (!ok && lane == 0) give_up(OZK_DEVERR_TIMEOUT_PRODUCER);
        if (PAIR && rank == 1 && lane == 0)
            st_cluster_u64(map_to_rank(smem_addr(const_cast<const long long*>(peer_issued)), 0u), (uint64_t)issued);
    } else if (warp == 1) {
        if (rank == 0) {
            // ------------------------------------------------------------ scales to TMEM, MMAs (the whole warp; one lane issues)
            int stage = 0, before = 0;
            uint32_t phase = 0, it = 0, step = 0;
            bool ok = true;
            const uint32_t tmem = (uint32_t)uniform((int)tmem_base);
            // descriptors: the address part advances with the stage, the rest is constant
            const uint64_t dL = umma_desc_sw128(smem_addr(sL)), dR = umma_desc_sw128(smem_addr(sR));
            const uint64_t dSL = smem_desc_scales(smem_addr(sSL)), dSR = smem_desc_scales(smem_addr(sSR));
            for (long long u = u0; ok && u < work.units; u += du) {
                const int b = (int)(it & 1u);
                if (it >= (uint32_t)S::LAG) {
                    const uint32_t bar = S::LAG == 1 ? acce_bar(0) : acce_bar(b);
                    const uint32_t par = S::LAG == 1 ? (it - 1u) & 1u : ((it >> 1) - 1u) & 1u;
                    ok = mbar_wait_warp(bar, par, abort_flag, a.limit_ns);
                    if (!ok) break;
                    tc_fence_after();
                }
                const uint32_t d_tmem = tmem + (uint32_t)(b * S::ACC_STRIDE);
                auto columns = [&](uint32_t st) { return tmem + (uint32_t)(S::SCALE_BASE + (int)(st & 1u) * S::SCALE_COLS); };
                // the four instructions of a stage: 32 bytes along K inside the swizzle atom each (+2 in the >> 4 address
                // field); the last stage of an odd number of scale tiles has half of them
                auto multiply = [&](int sg, uint32_t st, int kb) {
                    const uint64_t ld = dL + (uint64_t)(sg * (S::L_BYTES >> 4)), rd = dR + (uint64_t)(sg * (S::R_BYTES >> 4));
                    const uint32_t tl = columns(st), tr = tl + (uint32_t)(4 * S::KT);
                    const int tiles = min(S::KT, a.ktiles - kb * S::KT);
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) {
                        const int t = KIND == MXF4 ? kk >> 1 : 0;
                        if (t >= tiles) break;
                        const uint32_t idesc = a.idesc | umma_idesc_scale_id(KIND == MXF4 ? 2u * (kk & 1) : (uint32_t)kk);
                        const uint32_t acc = (kb > kb0 || kk > 0) ? 1u : 0u;
                        const uint32_t ca = tl + 4u * t, cb = tr + 4u * (uint32_t)(t * S::SUBS);
                        if (KIND == MXF4 && PAIR) umma_mxf4_pair(d_tmem, ld + 2u * kk, rd + 2u * kk, idesc, ca, cb, acc);
                        else if (KIND == MXF4) umma_mxf4(d_tmem, ld + 2u * kk, rd + 2u * kk, idesc, ca, cb, acc);
                        else if (PAIR) umma_mxf8f6f4_pair(d_tmem, ld + 2u * kk, rd + 2u * kk, idesc, ca, cb, acc);
                        else umma_mxf8f6f4(d_tmem, ld + 2u * kk, rd + 2u * kk, idesc, ca, cb, acc);
                    }
                    commit(empty_bar(sg));
                };
                for (int kb = kb0; kb < kb1; kb++) {
                    ok = mbar_wait_warp(full_bar(stage), phase, abort_flag, a.limit_ns);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t tl = columns(step), tr = tl + (uint32_t)(4 * S::KT);
                        const uint64_t sl = dSL + (uint64_t)(stage * (S::SL_BYTES >> 4)), sr = dSR + (uint64_t)(stage * (S::SR_BYTES >> 4));
#pragma unroll
                        for (int t = 0; t < S::KT; t++) {
                            if (PAIR) tmem_cp_scales_pair(tl + 4u * t, sl + (uint64_t)(t * (TILE_BYTES >> 4)));
                            else tmem_cp_scales(tl + 4u * t, sl + (uint64_t)(t * (TILE_BYTES >> 4)));
#pragma unroll
                            for (int i = 0; i < S::SUBS; i++) {
                                const uint64_t from = sr + (uint64_t)((i * S::SL_BYTES + t * TILE_BYTES) >> 4);
                                const uint32_t to = tr + 4u * (uint32_t)(t * S::SUBS + i);
                                if (PAIR) tmem_cp_scales_pair(to, from);
                                else tmem_cp_scales(to, from);
                            }
                        }
                        if (kb > kb0) multiply(before, step - 1u, kb - 1);
                    }
                    __syncwarp();
                    before = stage;
                    step++;
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
                if (!ok) break;
                if (elect_one()) {
                    multiply(before, step - 1u, kb1 - 1);
                    commit(accf_bar(b));
                }
                __syncwarp();
                it++;
            }
            if (!ok && lane == 0) give_up(OZK_DEVERR_TIMEOUT_MMA);
        }
    } else {
        // ---------------------------------------------------------------- epilogue warps
        const int ew = warp - 2;
        const int quarter = warp & 3;          // TMEM lanes this warp may access: [32 quarter, 32 quarter + 32)
        const int half = ew >> 2;              // column half of the accumulator
        constexpr int NCH = S::HALF / CHUNK;
        uint32_t it = 0;
        bool ok = true;
        auto drained = [&](int b) {            // one arrival a warp, on the barrier that the issuing CTA waits for
            if (PAIR) mbar_arrive_cluster(map_to_rank(acce_bar(b), 0u));
            else mbar_arrive(acce_bar(b));
        };
        for (long long u = u0; ok && u < work.units; u += du) {
            const Unit w = work.at(u);
            const int b = (int)(it & 1u);
            if (!mbar_wait_warp(accf_bar(b), (it >> 1) & 1u, abort_flag, a.limit_ns)) {
                if (lane == 0) give_up(OZK_DEVERR_TIMEOUT_EPILOGUE);
                ok = false;
                break;
            }
            __syncwarp();
            tc_fence_after();
            const int l = w.l0 + rank * BM + quarter * 32 + lane;
            const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * S::ACC_STRIDE + half * S::HALF);
            const int r = w.r0 + half * S::HALF;
            if (!PAIR && parts > 1) {
                float* mine = reinterpret_cast<float*>(smem);
#pragma unroll 1
                for (int c = 0; c < NCH; c++) {
                    uint32_t v[CHUNK];
                    tmem_ld_chunk<CHUNK>(acc + (uint32_t)(c * CHUNK), v);
                    tmem_wait_ld();
                    const int row = quarter * 32 + lane, col = half * S::HALF + c * CHUNK;
                    if (SWAP) {                // [column][row]: rows are neighbours in C
#pragma unroll
                        for (int e = 0; e < CHUNK; e++) mine[(col + e) * BM + row] = __uint_as_float(v[e]);
                    } else {                   // [row][column], four words of padding
#pragma unroll
                        for (int e = 0; e < CHUNK; e += 4)
                            *reinterpret_cast<uint4*>(mine + row * (BN + 4) + col + e) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                    }
                }
            } else if constexpr (SWAP) {
#pragma unroll 1
                for (int c = 0; c < NCH; c++) {
                    uint32_t v[CHUNK];
                    tmem_ld_chunk<CHUNK>(acc + (uint32_t)(c * CHUNK), v);
                    tmem_wait_ld();
                    if (c == NCH - 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) drained(b);
                    }
                    store_chunk<CHUNK, true>(a, w, l, r + c * CHUNK, v);
                }
            } else {
                // blocks of 64 columns.  Accumulators that overlap: those with the shared columns (the last 48 of buffer 0,
                // the first 48 of buffer 1) are read first, and a warp without them has nothing that the next tile waits for
                constexpr int BLOCKS = S::HALF / 64;
                const bool shared_half = S::LAG == 2 || half == 1 - b;
                const bool backward = S::LAG == 1 && b == 0;
                if (!shared_half && lane == 0) drained(0);
#pragma unroll 1
                for (int c = 0; c < BLOCKS; c++) {
                    const int at = (backward ? BLOCKS - 1 - c : c) * 64;
                    uint32_t v0[32], v1[32];
                    tmem_ld_32x32b_x32(acc + (uint32_t)at, v0);
                    tmem_ld_32x32b_x32(acc + (uint32_t)(at + 32), v1);
                    tmem_wait_ld();
                    if (shared_half && c == (S::LAG == 1 ? 0 : BLOCKS - 1)) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) drained(S::LAG == 1 ? 0 : b);
                    }
                    store_block<S::BOXES>(a, &tmC, w, l - lane, r + at, lane, smem_addr(sOut + ew * OUT_WARP_BYTES), v0, v1);
                }
                tc_fence_before();
                __syncwarp();
            }
            it++;
        }
        if (S::BOXES && lane == 0) bulk_wait_all();
        // rows of C behind the last group
        if (a.groups && a.fill) {
            const int size = a.dtype == OZK_F32 ? 4 : 2;
            const long long bytes = (long long)a.n * size;
            for (long long row = (long long)bound[a.groups] + blockIdx.x; row < a.tokens; row += gridDim.x) {
                uint8_t* p = static_cast<uint8_t*>(a.C) + row * a.ldc * size;
                const long long vecs = a.vec ? bytes / 16 : 0;
                for (long long i = threadIdx.x - 64; i < vecs; i += EPI_WARPS * 32)
                    reinterpret_cast<uint4*>(p)[i] = make_uint4(0u, 0u, 0u, 0u);
                for (long long i = vecs * 8 * 2 / size + threadIdx.x - 64; i < a.n; i += EPI_WARPS * 32)
                    store1(p, i, 0.0f, a.dtype);
            }
        }
    }

    if (!PAIR && parts > 1) {
        // add one slice of the tile over the cluster, four values a thread, CTA 0's sums first
        __syncwarp();
        cluster_sync();
        if (warp >= 2 && u0 < work.units && !*abort_flag) {
            const Unit w = work.at(u0);
            constexpr int LINE = SWAP ? BM : BN, LINES = SWAP ? BN : BM, PITCH = SWAP ? BM : BN + 4;
            constexpr int QUADS = LINES * LINE / 4;
            const uint32_t base = smem_addr(smem);
            for (int q = QUADS * part / parts + (int)threadIdx.x - 64; q < QUADS * (part + 1) / parts; q += EPI_WARPS * 32) {
                const int line = q / (LINE / 4), at = q % (LINE / 4) * 4;
                const uint32_t addr = base + 4u * (uint32_t)(line * PITCH + at);
                const int token = (SWAP ? w.r0 : w.l0) + line, col = (SWAP ? w.l0 : w.r0) + at;
                if (token < w.first || token >= w.last || col >= a.n) continue;
                float4 f[8];
#pragma unroll
                for (int p = 0; p < 8; p++)
                    if (p < parts) f[p] = ld_cluster_f32x4(map_to_rank(addr, (uint32_t)p));
                float4 s = f[0];
#pragma unroll
                for (int p = 1; p < 8; p++)
                    if (p < parts) { s.x += f[p].x; s.y += f[p].y; s.z += f[p].z; s.w += f[p].w; }
                store4(a, token, col, s);
            }
        }
        __syncwarp();
        cluster_sync();                        // no CTA leaves while another reads its sums
    }
    if (PAIR) {
        __syncwarp();
        cluster_sync();                        // nor while its peer's MMAs or arrivals still reach it
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (__builtin_expect(*abort_flag, 0)) {
        // All roles of the CTA (of the pair) have left, by a wait that ran out or at their end.  What they issued still writes
        // shared memory, TMEM and barriers, so it has to land before those are given up.
        if (warp == 0 && rank == 0) {
            if (lane == 0) drain_loads<STAGES>(issued, PAIR ? *peer_issued : issued, a.load_bytes, full_bar, DRAIN_LIMIT_NS);
        } else if (warp == 1) {
            if (rank == 0 && elect_one()) commit(drain_bar);
            __syncwarp();
            int none = 0;
            mbar_wait_bounded(drain_bar, 0u, &none, DRAIN_LIMIT_NS);
        }
        __syncwarp();
        if (PAIR) cluster_sync();
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    }
    if (warp == 1) {
        __syncwarp();
        if (PAIR) tmem_dealloc_pair(tmem_base, S::TMEM_COLS);
        else tmem_dealloc(tmem_base, S::TMEM_COLS);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn find_encode_fn() {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
        return reinterpret_cast<EncodeTiledFn>(p);
    return nullptr;
}

struct Operand {
    const uint8_t *codes, *scales;
    int fmt, groups, rows;
};

bool spreads(const Operand& o, int kind) { return kind == MXF8F6F4 && o.fmt == OZK_MX_E2M1; }

// codes [groups][rows][kp], box of 128 bytes of K (after the spreading of 4-bit codes, where `spread`) x box_rows rows,
// 128-byte swizzle; rows past the end are zero
int make_map(CUtensorMap* map, const Operand& o, int k, int box_rows, int kind) {
    static const EncodeTiledFn fn = find_encode_fn();
    if (!fn) return OZK_ERR_DRIVER;
    const bool spread = spreads(o, kind);
    const cuuint64_t pitch = (cuuint64_t)code_pitch(o.fmt, k);
    const cuuint64_t dims[3] = {spread ? (cuuint64_t)padded_k(k) : pitch, (cuuint64_t)o.rows, (cuuint64_t)o.groups};
    const cuuint64_t strides[2] = {pitch, pitch * (cuuint64_t)o.rows};
    const cuuint32_t box[3] = {(cuuint32_t)ROW_BYTES, (cuuint32_t)box_rows, 1u};
    const cuuint32_t estr[3] = {1u, 1u, 1u};
    const CUresult r = fn(map, spread ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3,
                          const_cast<uint8_t*>(o.codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? OZK_OK : OZK_ERR_DRIVER;
}

// scales [groups][row tiles][k tiles][512], box of KT k tiles x `tiles` row tiles; tiles past the end are zero
int make_scale_map(CUtensorMap* map, const Operand& o, int k, int kt, int tiles) {
    static const EncodeTiledFn fn = find_encode_fn();
    if (!fn) return OZK_ERR_DRIVER;
    const cuuint64_t ktiles = (cuuint64_t)(padded_k(k) / TILE), rtiles = (cuuint64_t)row_tiles(o.rows);
    const cuuint64_t dims[4] = {TILE_BYTES / 4, ktiles, rtiles, (cuuint64_t)o.groups};
    const cuuint64_t strides[3] = {TILE_BYTES, TILE_BYTES * ktiles, TILE_BYTES * ktiles * rtiles};
    const cuuint32_t box[4] = {TILE_BYTES / 4, (cuuint32_t)kt, (cuuint32_t)tiles, 1u};
    const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, const_cast<uint8_t*>(o.scales), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? OZK_OK : OZK_ERR_DRIVER;
}

// C: boxes of 32 rows x 128 bytes, 128-byte swizzle
int make_out_map(CUtensorMap* map, const Args& a) {
    static const EncodeTiledFn fn = find_encode_fn();
    if (!fn) return OZK_ERR_DRIVER;
    const cuuint64_t size = a.dtype == OZK_F32 ? 4 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t)a.n, (cuuint64_t)a.tokens};
    const cuuint64_t strides[1] = {(cuuint64_t)a.ldc * size};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / size), 32u};
    const cuuint32_t estr[2] = {1u, 1u};
    const CUresult r = fn(map, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, a.C, dims,
                          strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? OZK_OK : OZK_ERR_DRIVER;
}

// SM count of the current device, 0 when it is not a B200
int sm_count(int* dev_out) {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int sms = known[dev].load(std::memory_order_relaxed);
    if (sms == 0) {
        int major = 0;
        if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10) return 0;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        known[dev].store(sms, std::memory_order_relaxed);
    }
    *dev_out = dev;
    return sms;
}

struct Call {
    Operand A, B;
    int n, k, kind;
    Args args;
    cudaStream_t st;
    int dev, sms;
    bool hold;                               // self-test: expect more of every stage than its loads bring
};

uint32_t format_bits(int kind, int fmt) { return kind == MXF4 ? 1u : fmt == OZK_MX_E2M1 ? 5u : 0u; }

template <int KIND, int BN, bool SWAP, bool PAIR>
int launch(const Call& c, int parts) {
    using S = Shape<KIND, BN, SWAP, PAIR>;
    auto kern = mx_gemm_kernel<KIND, BN, SWAP, PAIR>;
    const Operand &L = SWAP ? c.B : c.A, &R = SWAP ? c.A : c.B;
    Args a = c.args;
    a.l_rows = L.rows;
    a.r_rows = R.rows;
    a.ktiles = padded_k(c.k) / TILE;
    a.kblocks = (a.ktiles + S::KT - 1) / S::KT;
    // a load that spreads 4-bit codes counts the bytes it reads, not the bytes it fills
    a.load_bytes = S::L_BYTES / (spreads(L, KIND) ? 2u : 1u) + S::R_BYTES / (spreads(R, KIND) ? 2u : 1u) + S::SL_BYTES + S::SR_BYTES +
                   (c.hold ? 16u : 0u);
    a.idesc = umma_idesc_mx(format_bits(KIND, L.fmt), format_bits(KIND, R.fmt), S::BL, BN);
    CUtensorMap tl, tr, tsl, tsr, tc = {};
    int rc;
    if ((rc = make_map(&tl, L, c.k, BM, KIND)) != OZK_OK) return rc;
    if ((rc = make_map(&tr, R, c.k, S::RN, KIND)) != OZK_OK) return rc;
    if ((rc = make_scale_map(&tsl, L, c.k, S::KT, 1)) != OZK_OK) return rc;
    if ((rc = make_scale_map(&tsr, R, c.k, S::KT, S::SUBS)) != OZK_OK) return rc;
    if (S::BOXES && parts == 1 && a.vec && (rc = make_out_map(&tc, a)) != OZK_OK) return rc;
    const long long lt = (L.rows + S::BL - 1) / S::BL, rt = (R.rows + BN - 1) / BN;
    if (lt * rt > 0x7fffffffLL || (SWAP && rt > 1)) return OZK_ERR_ARG;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute cluster[1];
    cluster[0].id = cudaLaunchAttributeClusterDimension;
    cluster[0].val.clusterDim.x = (unsigned)(PAIR ? 2 : parts);
    cluster[0].val.clusterDim.y = 1;
    cluster[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = c.st;
    cfg.attrs = cluster;
    cfg.numAttrs = PAIR || parts > 1 ? 1 : 0;
    // once per device: the shared memory limit, and for pairs how many fit at once
    static std::atomic<int> resident[64];
    int fit = resident[c.dev].load(std::memory_order_acquire);
    if (fit == 0) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
        if (e != cudaSuccess) return OZK_ERR_CUDA_BASE + (int)e;
        fit = c.sms;
        if (PAIR) {
            cfg.gridDim = dim3((unsigned)(c.sms / 2 * 2), 1, 1);
            e = cudaOccupancyMaxActiveClusters(&fit, kern, &cfg);
            if (e != cudaSuccess) return OZK_ERR_CUDA_BASE + (int)e;
            if (fit < 1) return OZK_ERR_DEVICE;
        }
        resident[c.dev].store(fit, std::memory_order_release);
    }
    // grouped: the number of tiles is known on the device only
    const long long units = a.groups ? fit : lt * rt;
    const long long grid = PAIR ? 2 * (units < fit ? units : fit) : parts > 1 ? units * parts : units < fit ? units : fit;
    cfg.gridDim = dim3((unsigned)grid, 1, 1);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tl, tr, tsl, tsr, tc, a, parts);
    if (e != cudaSuccess) return OZK_ERR_CUDA_BASE + (int)e;
    OZK_CHECK_LAUNCH();
    return OZK_OK;
}

// CTAs that share one tile along K: as many as keep the grid within the SMs, with at least `least` stages each
int parts_for(long long units, int kblocks, int sms, int least) {
    int p = 1;
    while (p < 8 && units * p * 2 <= sms && kblocks >= 2 * p * least) p *= 2;
    return p;
}

// Which tile.  Every stage costs about 0.25 us whatever the tile's width, so wide tiles win as soon as they fill the SMs,
// and where they do not, K is split.  Measured, us (e4m3 x e4m3, n = k = 4096; in brackets e2m1 x e2m1):
//   m = 16:   B left, 32 rows of A, K in four 7.7 (6.8); 64 rows 8.9 (7.5); 128 x 128 in four 10.8 (8.8); pair 15.0 (10.4)
//   m = 64:   B left, 64 rows, K in four 8.8 (7.5); 128 x 128 in four 9.7 (8.1)
//   m = 128:  128 x 128 in four 10.1 (8.7), unsplit 15.0 (10.1); B left, 64 rows, in two 11.6 (9.1); pair 15.6 (11.2)
//   m = 512:  128 x 128 16.5 (10.8); pair 16.1 (11.4)
//   m = 768:  pair 16.5 (11.7); 128 x 128 (192 tiles, more than SMs) 26.3 (16.1)
// with n = 65536 (e4m3 x e2m1): m = 16: B left 45, 128 x 256 50; m = 64: 47, 42; m = 128: 128 x 128 or pair 64, 128 x 256 45;
// and with n = k = 1024, where the split's exchange costs more than it saves: m = 512 unsplit 7.3 (6.3), in four 8.0 (7.6).
// Grouped, 16 experts of 4096 x 2048 in e2m1, A in e4m3 (in brackets e2m1), by the rows of an average group:
//   8: 128 x 256 22.6 (15.6), pair 31.8 (23.9); 32: 30.0 (19.3), 32.3 (23.7); 64: 35.8 (21.6), 33.6 (23.7);
//   100: 46.0 (26.8), 35.3 (24.4); 256: 73.1 (44.6), 53.6 (37.8); 1024: 181 (107), 138 (90).
// (The 4-bit kind does better with the smaller tile for a little longer: by 6 % at m = 512, by 9 % at groups of 64 rows.  It
// has no rule of its own.)  For 65 to 128 rows and n from 128 to 384 times the SMs the pair runs with its second 128
// rows empty; only n = 65536, where 128 x 256 won, was measured.
// Rows of C off 16-byte boundaries leave value by value: 4096 x 50257 x 1024 in e4m3 takes 1995 us, 4096 x 50256 x 1024 221.
template <int KIND>
int choose(const Call& c) {
    const int kblocks = (padded_k(c.k) / TILE + (KIND == MXF4 ? 1 : 0)) / (KIND == MXF4 ? 2 : 1);
    if (c.args.groups) {
        if (c.args.tokens / c.args.groups < 64) return launch<KIND, 256, false, false>(c, 1);
        return launch<KIND, 256, false, true>(c, 1);
    }
    const long long m = c.A.rows, nt = (c.n + BM - 1) / BM, squares = ((m + BM - 1) / BM) * nt;
    if (m > 32 && m <= 128 && c.n >= 384LL * c.sms) return launch<KIND, 256, false, false>(c, 1);
    if (m <= 64 && kblocks >= 8) {
        const int parts = parts_for(nt, kblocks, c.sms, 2);
        return m <= 32 ? launch<KIND, 32, true, false>(c, parts) : launch<KIND, 64, true, false>(c, parts);
    }
    if (squares <= c.sms) return launch<KIND, 128, false, false>(c, kblocks >= 16 ? parts_for(squares, kblocks, c.sms, 4) : 1);
    return launch<KIND, 256, false, true>(c, 1);
}

int run(const uint8_t* Ac, const uint8_t* As, int Af, const uint8_t* Bc, const uint8_t* Bs, int Bf, int m, int n, int k,
        int groups, const int32_t* ends, int fill, void* C, int64_t ldc, int dtype, int32_t* err, ozk_stream_t stream,
        uint64_t limit_ns = WAIT_LIMIT_NS, bool hold = false) {
    if (!Ac || !As || !Bc || !Bs || !C || !err || !fmt_ok(Af) || !fmt_ok(Bf)) return OZK_ERR_ARG;
    if (m < 1 || n < 1 || m > OZK_MX_ROWS_MAX || n > OZK_MX_ROWS_MAX || k < 1 || k > OZK_MX_KMAX || ldc < n) return OZK_ERR_ARG;
    if (!dtype_ok(dtype)) return OZK_ERR_ARG;
    const uintptr_t align = reinterpret_cast<uintptr_t>(Ac) | reinterpret_cast<uintptr_t>(Bc);
    const uintptr_t align_s = reinterpret_cast<uintptr_t>(As) | reinterpret_cast<uintptr_t>(Bs);
    const uintptr_t size = dtype == OZK_F32 ? 4 : 2;
    if ((align & 31) || (align_s & 15) || (reinterpret_cast<uintptr_t>(C) & (size - 1))) return OZK_ERR_ARG;
    Call c;
    c.sms = sm_count(&c.dev);
    if (c.sms == 0) return OZK_ERR_DEVICE;
    c.A = {Ac, As, Af, 1, m};
    c.B = {Bc, Bs, Bf, groups ? groups : 1, n};
    c.n = n;
    c.k = k;
    c.kind = Af == OZK_MX_E2M1 && Bf == OZK_MX_E2M1 ? MXF4 : MXF8F6F4;
    c.st = reinterpret_cast<cudaStream_t>(stream);
    c.hold = hold;
    Args& a = c.args;
    a = Args{};
    a.groups = groups;
    a.ends = ends;
    a.tokens = m;
    a.n = n;
    a.fill = fill;
    a.C = C;
    a.ldc = ldc;
    a.dtype = dtype;
    // (a tensor map's stride ends at 2^40 bytes)
    a.vec = (reinterpret_cast<uintptr_t>(C) & 15) == 0 && ldc * (int64_t)size % 16 == 0 && ldc < ((int64_t)1 << 37);
    a.err = err;
    a.limit_ns = limit_ns;
    return c.kind == MXF4 ? choose<MXF4>(c) : choose<MXF8F6F4>(c);
}

}  // namespace

extern "C" int ozk_mx_gemm(const uint8_t* A_codes, const uint8_t* A_scales, int A_fmt, const uint8_t* B_codes,
                           const uint8_t* B_scales, int B_fmt, int m, int n, int k, void* C, int64_t ldc, int dtype,
                           int32_t* err, ozk_stream_t stream) {
    return run(A_codes, A_scales, A_fmt, B_codes, B_scales, B_fmt, m, n, k, 0, nullptr, 0, C, ldc, dtype, err, stream);
}

extern "C" int ozk_mx_grouped_gemm(const uint8_t* A_codes, const uint8_t* A_scales, int A_fmt, const uint8_t* B_codes,
                                   const uint8_t* B_scales, int B_fmt, int rows, int n, int k, int groups,
                                   const int32_t* ends, int fill, void* C, int64_t ldc, int dtype, int32_t* err,
                                   ozk_stream_t stream) {
    if (!ends || (reinterpret_cast<uintptr_t>(ends) & 3) || groups < 1 || groups > OZK_MX_MAX_GROUPS) return OZK_ERR_ARG;
    return run(A_codes, A_scales, A_fmt, B_codes, B_scales, B_fmt, rows, n, k, groups, ends, fill, C, ldc, dtype, err,
               stream);
}

extern "C" int ozk_mx_wait_selftest(const uint8_t* A_codes, const uint8_t* A_scales, int A_fmt, const uint8_t* B_codes,
                                    const uint8_t* B_scales, int B_fmt, int m, int n, int k, void* C, int64_t ldc, int dtype,
                                    int64_t limit_ns, int hold, int32_t* err, ozk_stream_t stream) {
    if (limit_ns < 100 || limit_ns > (int64_t)WAIT_LIMIT_NS) return OZK_ERR_ARG;
    return run(A_codes, A_scales, A_fmt, B_codes, B_scales, B_fmt, m, n, k, 0, nullptr, 0, C, ldc, dtype, err, stream,
               (uint64_t)limit_ns, hold != 0);
}
