// Root-mean-square norm with the residual's addition that writes an MX operand for the next product.
#include <math.h>

#include "mx_common.cuh"

using namespace ozk_mx;

namespace {

// ---- root-mean-square norm with an MX output -----------------------------------------------------------------------
// t = x (+ residual), y = t / sqrt(mean(t^2) + eps) weight, y quantised; t, rounded to the type of x, is the next
// residual.  Everything between the loads and the codes stays in registers: one pass over x and the residual, TPR threads
// a row with NC chunks of eight values each (longer rows read the rest a second time).  The sums are taken in a fixed
// order; the inverse root is rounded once, t times the root (at most sqrt(d), so it never overflows) and its product with
// the weight once each.
// Sum over the threads of a row: a warp's in FP32, the warps' in FP64.  `part` is free again after the block's next barrier.
template <int TPR>
__device__ __forceinline__ double row_sum(float share, double* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) share += __shfl_xor_sync(0xffffffffu, share, o);
    if (TPR == 32) return (double)share;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = (double)share;
    __syncthreads();
    double v = (threadIdx.x & 31) < TPR / 32 ? part[threadIdx.x & 31] : 0.0;
#pragma unroll
    for (int o = TPR / 64; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0);
}

// Rows whose sum of squares and eps are beyond FP32 (or NaN) take their squares again of t 2^-80 (a warp adds up to 2^23 of
// them, each up to 2^96), and are normed as t / 16 and 16 / sqrt(mean t^2 + eps): the root itself would be subnormal for the
// largest t.
__device__ __forceinline__ bool beyond_f32(double total, float eps) { return !(total + (double)eps < 3.0e38); }

// 1 / sqrt(a) to the nearest FP32 number or its neighbour, for a below 3e38: FP32's root and one Newton step with an exact
// residual 1 - a r^2
__device__ __forceinline__ float inverse_root(double a) {
    const float ah = (float)a, al = (float)(a - (double)ah);
    const float r = rsqrtf(ah);
    const float q = ah * r, qe = fmaf(ah, r, -q);
    const float e = fmaf(-q, r, 1.0f) - fmaf(qe, r, al * r * r);
    return fmaf(0.5f * r, e, r);
}

// Eight normed values of a row (chunk c) to codes and, from the first of the 16 lanes that hold a k tile, its four scale
// bytes; called by whole warps (the chunks of a row are a multiple of 16, so those lanes are all in or all out)
template <int FMT>
__device__ __forceinline__ void emit_chunk(float (&o)[8], bool up, int c, bool in, uint8_t* __restrict__ cr,
                                           uint8_t* __restrict__ tr) {
    const int s = block_scale<FMT>(quad_max(max_bits8(o)), up);
    const float inv = scale_inverse(s);
#pragma unroll
    for (int j = 0; j < 8; j++) o[j] *= inv;
    const uint2 e = encode8<FMT>(o, s == 255);
    if (in) {
        if (FMT == OZK_MX_E2M1)
            *reinterpret_cast<uint32_t*>(cr + c * 4) = e.x;
        else
            *reinterpret_cast<uint2*>(cr + c * 8) = e;
    }
    uint32_t four = (uint32_t)s;
    four |= __shfl_down_sync(0xffffffffu, four, 4) << 8;
    four |= __shfl_down_sync(0xffffffffu, four, 8) << 16;
    if (in && (c & 15) == 0) *reinterpret_cast<uint32_t*>(tr + (long long)(c / 16) * TILE_BYTES) = four;
}

// Eight neighbouring values as they lie in memory: unit c of a row, the 8 sizeof(T) bytes x c behind the 16-byte boundary at
// or before its first value, holds the values from 8 c - lead on (lead: the values between the boundary and the row).
template <typename T>
struct Raw8 {
    static constexpr int NG = sizeof(T) / 2;
    uint4 w[NG];
    // vectors from the row's end on are zero; those that pass the matrix's end are read value by value
    __device__ __forceinline__ void load(uintptr_t unit, uintptr_t row_end, uintptr_t end) {
#pragma unroll
        for (int i = 0; i < NG; i++) w[i] = load_granule(unit + 16 * i, row_end, 0, end);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < NG; i++) {
                v[4 * i] = __uint_as_float(w[i].x); v[4 * i + 1] = __uint_as_float(w[i].y);
                v[4 * i + 2] = __uint_as_float(w[i].z); v[4 * i + 3] = __uint_as_float(w[i].w);
            }
        } else {
            const uint32_t e[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = unpack2(e[j], (const T*)nullptr);
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
        }
    }
};

// The eight values of a chunk (from 8 c on) out of the units c (`v`) and c + 1: the next lane's, or for a warp's last lane
// the ones that the next warp left in `edge`
template <int LEAD>
__device__ __forceinline__ void take_chunk(float (&v)[8], const float* edge, bool last) {
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (j + LEAD < 8) {
            o[j] = v[(j + LEAD) & 7];
        } else {
            const float n = __shfl_down_sync(0xffffffffu, v[(j + LEAD) & 7], 1);
            o[j] = last ? edge[(j + LEAD) & 7] : n;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = o[j];
}

// Eight values of type T kept in as few registers as they need
template <typename T>
struct Kept8 {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 2 * (int)sizeof(T); j++) {
            if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[j]);
            else w[j] = pack2(v[2 * j], v[2 * j + 1], (const T*)nullptr);
        }
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[j]);
        } else {
            const float2 f = unpack2(w[j / 2], (const T*)nullptr);
            return j & 1 ? f.y : f.x;
        }
    }
};

// Many rows that fit into the registers of TPR threads (NC units of eight values each): CTAs stay and take rows in turn, with
// the next row's loads under way while a row is summed and encoded, and the weights in registers.  Rows need not start on
// 16 bytes (`SHIFTED`), as long as those of x, residual and sum do so alike: everything up to the sum of squares and the
// new residual happens in units of memory, and only then do the values move by `lead` places to where their blocks of 32
// begin.  bf16 16384 x 8192 with the residual to e4m3: 148 us, 6.3 TB/s (264 us with a CTA a row); to e2m1 145; bf16 8192 x
// 4097: 80 us (153).
// CTAs an SM: 1024 threads with 64 registers, 768 with 85 for three units a thread.  FP32 rows, and FP32 weights of 16-bit
// rows, do not fit there with two units or more a thread and spill (16-bit rows up to 160 bytes, FP32 up to 760): FP32 8192 x
// 8192 with the residual 144 - 154 us, 5.7 - 6.1 TB/s; 8192 x 5120, three units, 111 us, 4.9 TB/s.
constexpr int stream_blocks(int tpr, int nc) { return (nc > 2 ? 768 : 1024) / tpr; }

template <typename T, typename W, int FMT, int TPR, int NC, bool SHIFTED>
__global__ void __launch_bounds__(TPR, stream_blocks(TPR, NC))
    rms_norm_stream_kernel(const T* __restrict__ x, long long x_stride, const T* __restrict__ residual, long long res_stride,
                           const W* __restrict__ weight, int rows, int d, double inv_d, float eps, bool weight_aligned, bool up,
                           T* __restrict__ sum, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    __shared__ double part[2][32];
    __shared__ __align__(16) float edge[SHIFTED ? 2 : 1][SHIFTED ? NC : 1][SHIFTED ? TPR / 32 + 1 : 1][8];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, chunks = padded_k(d) / 8;
    Raw8<T> rx[NC], rr[NC];
    Kept8<W> w[NC];
    const uintptr_t x_end = reinterpret_cast<uintptr_t>(x + (rows - 1) * x_stride + d);
    const uintptr_t r_end = reinterpret_cast<uintptr_t>(residual + (rows - 1) * res_stride + d);
    auto fetch = [&](int row) {
        const uintptr_t px = reinterpret_cast<uintptr_t>(x + row * x_stride), pr = reinterpret_cast<uintptr_t>(residual + row * res_stride);
        const uintptr_t bytes = (uintptr_t)d * sizeof(T);
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const uintptr_t at = (uintptr_t)(t + i * TPR) * (8 * sizeof(T));
            rx[i].load((px & ~(uintptr_t)15) + at, px + bytes, x_end);
            if (residual) rr[i].load((pr & ~(uintptr_t)15) + at, pr + bytes, r_end);
        }
    };
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const int col = (t + i * TPR) * 8;
        float u[8];
        load8(weight + col, weight_aligned && col + 8 <= d, max(0, d - col), u);
        w[i].set(u);
    }
    if (SHIFTED && t < 16) edge[t / 8][NC - 1][TPR / 32][t & 7] = 0.0f;   // behind the last unit, which no warp writes
    fetch(blockIdx.x);
    const long long pitch = code_pitch(FMT, d);
    int turn = 0;
    for (int row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
        const int lead = SHIFTED ? (int)((reinterpret_cast<uintptr_t>(x + row * x_stride) & 15) / sizeof(T)) : 0;
        float v[NC][8];
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; i++) {
            rx[i].get(v[i]);
            if (residual) {
                float q[8];
                rr[i].get(q);
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] += q[j];
            }
            const int k = (t + i * TPR) * 8 - lead;             // the row's value that the unit begins with
            if (k < 0 || k + 8 > d) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (k + j < 0 || k + j >= d) v[i][j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) sq = fmaf(v[i][j], v[i][j], sq);
        }
        if (row + (int)gridDim.x < rows) fetch(row + (int)gridDim.x);
        if (sum) {
            T* to = sum + row * (long long)d;
#pragma unroll
            for (int i = 0; i < NC; i++) {
                const int k = (t + i * TPR) * 8 - lead;
                if (k >= 0 && k + 8 <= d) {
                    store8(to + k, true, 8, v[i]);
                } else if (k + 8 > 0 && k < d) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (k + j >= 0 && k + j < d) to[k + j] = from_f32<T>(v[i][j]);
                }
            }
        }
        auto leave_edges = [&] {                                // for the last lane of the warp before
            if constexpr (SHIFTED) {
                if (lane != 0) return;
#pragma unroll
                for (int i = 0; i < NC; i++) {
                    const int slot = warp > 0 ? i : i - 1;
                    if (slot < 0) continue;
                    float4* e = reinterpret_cast<float4*>(edge[turn][slot][warp > 0 ? warp : TPR / 32]);
                    e[0] = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
                    e[1] = make_float4(v[i][4], v[i][5], v[i][6], v[i][7]);
                }
            }
        };
        leave_edges();
        double total = row_sum<TPR>(sq, part[turn]);
        float rstd;
        if (beyond_f32(total, eps)) {
            sq = 0.0f;
#pragma unroll
            for (int i = 0; i < NC; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float u = v[i][j] * 0x1p-80f;
                    sq = fmaf(u, u, sq);
                    v[i][j] *= 0.0625f;
                }
            leave_edges();
            __syncthreads();
            total = row_sum<TPR>(sq, part[turn]) * 0x1p160;
            rstd = (float)(16.0 / sqrt(total * inv_d + (double)eps));
        } else {
            rstd = inverse_root(total * inv_d + (double)eps);
        }
        if (SHIFTED) {
            auto shift = [&](auto take) {
#pragma unroll
                for (int i = 0; i < NC; i++) take(v[i], edge[turn][i][warp + 1], lane == 31);
            };
            switch (lead) {
                case 1: shift(take_chunk<1>); break;
                case 2: shift(take_chunk<2>); break;
                case 3: shift(take_chunk<3>); break;
                case 4: shift(take_chunk<4>); break;
                case 5: shift(take_chunk<5>); break;
                case 6: shift(take_chunk<6>); break;
                case 7: shift(take_chunk<7>); break;
                default: break;
            }
        }
        uint8_t* cr = codes + row * pitch;
        uint8_t* tr = scales + (row / TILE) * (long long)(chunks / 16) * TILE_BYTES + scale_slot(row % TILE, 0);
#pragma unroll
        for (int i = 0; i < NC; i++) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = v[i][j] * rstd * w[i].get(j);
            emit_chunk<FMT>(v[i], up, t + i * TPR, t + i * TPR < chunks, cr, tr);
        }
    }
}

template <typename T, typename W, int FMT, int TPR, int NC>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR, TPR == 32 ? 6 : 1024 / TPR)
    rms_norm_kernel(const T* __restrict__ x, long long x_stride, const T* __restrict__ residual, long long res_stride,
                    const W* __restrict__ weight, int rows, int d, double inv_d, float eps, bool aligned, bool up,
                    T* __restrict__ sum, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    __shared__ double part[32];
    constexpr int RPB = TPR == 32 ? 4 : 1;
    const long long row = (long long)blockIdx.x * RPB + (RPB == 1 ? 0 : threadIdx.x / TPR);
    const int t = RPB == 1 ? threadIdx.x : threadIdx.x % TPR;
    if (row >= rows) return;                                   // whole warps only (RPB > 1): no barrier follows them
    const int kp = padded_k(d), chunks = kp / 8;
    const T* xr = x + row * x_stride;
    const T* rr = residual ? residual + row * res_stride : nullptr;
    T* sr = sum ? sum + row * (long long)d : nullptr;

    float v[NC][8];
    auto fetch = [&](int c, float (&o)[8]) {
        const int col = c * 8;
        const bool whole = aligned && col + 8 <= d;
        const int count = max(0, d - col);
        load8(xr + col, whole, count, o);
        if (rr) {
            float q[8];
            load8(rr + col, whole, count, q);
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] += q[j];
        }
    };
    // sum of f(t)^2
    auto squares = [&](auto f, bool store) {
        float sq = 0.0f;
        auto note = [&](int c, const float (&o)[8]) {
            if (store && sr) store8(sr + c * 8, aligned && c * 8 + 8 <= d, max(0, d - c * 8), o);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float u = f(o[j]);
                sq = fmaf(u, u, sq);
            }
        };
#pragma unroll
        for (int i = 0; i < NC; i++)
            if (t + i * TPR < chunks) note(t + i * TPR, v[i]);
        for (int c = t + NC * TPR; c < chunks; c += TPR) {
            float o[8];
            fetch(c, o);
            note(c, o);
        }
        if (TPR > 32) __syncthreads();                         // `part` may still be read from an earlier sum
        return row_sum<TPR>(sq, part);
    };
#pragma unroll
    for (int i = 0; i < NC; i++)
        if (t + i * TPR < chunks) fetch(t + i * TPR, v[i]);
    double total = squares([](float x) { return x; }, true);
    float rstd, down = 1.0f;
    if (beyond_f32(total, eps)) {
        total = squares([](float x) { return x * 0x1p-80f; }, false) * 0x1p160;
        rstd = (float)(16.0 / sqrt(total * inv_d + (double)eps));
        down = 0.0625f;
#pragma unroll
        for (int i = 0; i < NC; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] *= down;
    } else {
        rstd = inverse_root(total * inv_d + (double)eps);
    }

    const long long pitch = code_pitch(FMT, d);
    uint8_t* cr = codes + row * pitch;
    uint8_t* tr = scales + (row / TILE) * (long long)(kp / TILE) * TILE_BYTES + scale_slot((int)(row % TILE), 0);
    auto emit = [&](int c, float (&o)[8], bool in) {
        float w[8];
        load8(weight + c * 8, in && aligned && c * 8 + 8 <= d, in ? max(0, d - c * 8) : 0, w);
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = in ? o[j] * rstd * w[j] : 0.0f;
        emit_chunk<FMT>(o, up, c, in, cr, tr);
    };
#pragma unroll
    for (int i = 0; i < NC; i++) emit(t + i * TPR, v[i], t + i * TPR < chunks);
    for (int c0 = NC * TPR; c0 < chunks; c0 += TPR) {           // the same trips for every lane of a warp
        const int c = c0 + t;
        float o[8] = {};
        if (c < chunks) fetch(c, o);
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] *= down;
        emit(c, o, c < chunks);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
struct NormArgs {
    const void *x, *residual, *weight;
    long long x_stride, res_stride;
    int rows, d;
    float eps;
    bool up;
    void* sum;
    uint8_t *codes, *scales;
    cudaStream_t st;
    int sms;
};

template <typename T, typename W, int FMT>
int launch_norm(const NormArgs& a) {
    const long long size = (long long)sizeof(T);
    const bool aligned = aligned16(a.x) && aligned16(a.residual) && aligned16(a.weight) && aligned16(a.sum) &&
                         (a.rows == 1 || (a.x_stride * size % 16 == 0 && (!a.residual || a.res_stride * size % 16 == 0) &&
                                          (!a.sum || a.d * size % 16 == 0)));
    // threads a row: enough that the values of up to 16384 stay in registers, a warp for short rows
    const int d = a.d;
#define OZK_NORM(TPR, NC)                                                                                            \
    rms_norm_kernel<T, W, FMT, TPR, NC>                                                                              \
        <<<(unsigned)((a.rows + (TPR == 32 ? 3 : 0)) / (TPR == 32 ? 4 : 1)), TPR == 32 ? 128 : TPR, 0, a.st>>>(      \
            static_cast<const T*>(a.x), a.x_stride, static_cast<const T*>(a.residual), a.res_stride,                 \
            static_cast<const W*>(a.weight), a.rows, d, 1.0 / d, a.eps, aligned, a.up, static_cast<T*>(a.sum), a.codes, a.scales)
#define OZK_STREAM(TPR, NC)                                                                                          \
    {                                                                                                                \
        auto kern = whole ? rms_norm_stream_kernel<T, W, FMT, TPR, NC, false>                                        \
                          : rms_norm_stream_kernel<T, W, FMT, TPR, NC, true>;                                        \
        const int grid = a.sms * stream_blocks(TPR, NC);                                                             \
        kern<<<(unsigned)(a.rows < grid ? a.rows : grid), TPR, 0, a.st>>>(                                           \
            static_cast<const T*>(a.x), a.x_stride, static_cast<const T*>(a.residual), a.res_stride,                 \
            static_cast<const W*>(a.weight), a.rows, d, 1.0 / d, a.eps, aligned16(a.weight), a.up,                   \
            static_cast<T*>(a.sum), a.codes, a.scales);                                                              \
    }
    // rows enough for every CTA to take several, and all three tensors' rows at the same place of their 16 bytes: the
    // streaming kernel (with rows that start anywhere, one unit more than the chunks of eight may be needed)
    const bool whole = aligned;
    const bool alike = aligned16(a.x) && aligned16(a.residual) && aligned16(a.sum) &&
                       (!a.residual || (a.res_stride - a.x_stride) * size % 16 == 0) &&
                       (!a.sum || (d - a.x_stride) * size % 16 == 0);
    const int need = d + (whole ? 0 : 8);
    if ((whole || alike) && d > 256 && need <= 16384 && a.rows >= 4 * a.sms) {
        if (need <= 1024) OZK_STREAM(128, 1)
        else if (need <= 2048) OZK_STREAM(256, 1)
        else if (need <= 4096) OZK_STREAM(256, 2)
        else if (need <= 6144) OZK_STREAM(256, 3)
        else if (need <= 8192) OZK_STREAM(512, 2)
        else OZK_STREAM(1024, 2)
    }
    else if (d <= 1024) OZK_NORM(32, 4);
    else if (d <= 2048) OZK_NORM(256, 1);
    else if (d <= 4096) OZK_NORM(256, 2);
    else if (d <= 8192) OZK_NORM(512, 2);
    else OZK_NORM(1024, 2);
#undef OZK_NORM
#undef OZK_STREAM
    OZK_CHECK_LAUNCH();
    return OZK_OK;
}

template <typename T>
int dispatch_norm(const NormArgs& a, bool weight_f32, int fmt) {
    if (fmt == OZK_MX_E2M1)
        return weight_f32 ? launch_norm<T, float, OZK_MX_E2M1>(a) : launch_norm<T, T, OZK_MX_E2M1>(a);
    return weight_f32 ? launch_norm<T, float, OZK_MX_E4M3>(a) : launch_norm<T, T, OZK_MX_E4M3>(a);
}

}  // namespace

extern "C" int ozk_mx_rms_norm(const void* x, const void* residual, const void* weight, int dtype, int weight_f32,
                               int rows, int d, int64_t x_stride, int64_t residual_stride, float eps, int fmt,
                               int round_up, void* sum, uint8_t* codes, uint8_t* scales, ozk_stream_t stream) {
    if (!x || !weight || !codes || !scales || !fmt_ok(fmt) || rows < 1 || rows > OZK_MX_ROWS_MAX || d < 1 ||
        d > OZK_MX_KMAX)
        return OZK_ERR_ARG;
    if (!(eps > 0.0f) || !(eps < INFINITY) || x_stride < 0 || residual_stride < 0) return OZK_ERR_ARG;
    if (!aligned16(codes) || !aligned16(scales)) return OZK_ERR_ARG;
    if (!dtype_ok(dtype) || !on_elements(x, dtype) || !on_elements(residual, dtype) || !on_elements(sum, dtype) ||
        !on_elements(weight, weight_f32 ? OZK_F32 : dtype))
        return OZK_ERR_ARG;
    int sms = 0;
    const int rc = ozk_device_sm_count(&sms);
    if (rc != OZK_OK) return rc;
    const NormArgs a = {x,    residual,      weight, x_stride, residual_stride, rows,
                        d,    eps,           round_up != 0,    sum,  codes,  scales,
                        reinterpret_cast<cudaStream_t>(stream), sms};
    if (dtype == OZK_F32) return dispatch_norm<float>(a, true, fmt);
    if (dtype == OZK_F16) return dispatch_norm<__half>(a, weight_f32 != 0, fmt);
    return dispatch_norm<__nv_bfloat16>(a, weight_f32 != 0, fmt);
}
