// Operand preparation for the microscaled products: quantisation to MX codes and scales, the way back, and the
// root-mean-square norm that writes an MX operand.
#include <math.h>

#include "mx_common.cuh"

using namespace ozk_mx;

namespace {

constexpr int THREADS = 256;

// ---- quantisation, contracted axis contiguous ----------------------------------------------------------------------
// One CTA per scale tile (128 rows x 128 elements): 16 lanes hold a row's 128 elements, eight each, so a block of 32 is
// four lanes and its largest magnitude two shuffles away.  All of a thread's eight loads are issued before the first is
// used.  The tile's 512 scale bytes are gathered in shared memory and leave as one contiguous store.
template <typename T, int FMT>
__global__ void __launch_bounds__(THREADS)
    quantize_rows_kernel(const T* __restrict__ x, long long group_stride, long long row_stride, int rows, int k,
                         bool up, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    __shared__ __align__(16) uint8_t sc[TILE_BYTES];
    const int ktiles = padded_k(k) / TILE, rtiles = row_tiles(rows);
    const int kt = (int)(blockIdx.x % (unsigned)ktiles);
    const int t = (int)(blockIdx.x / (unsigned)ktiles);
    const int rt = t % rtiles, g = t / rtiles;
    const int lane16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int col = kt * TILE + lane16 * 8;
    const int here = min(TILE, rows - rt * TILE);
    const T* xt = x + g * group_stride + (long long)rt * TILE * row_stride + col;
    const bool whole = col + 8 <= k;
    const int count = max(0, k - col);

    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = r0 + 16 * i;
        load8(xt + (long long)r * row_stride, whole && r < here, r < here ? count : 0, v[i]);
    }
    const long long pitch = code_pitch(FMT, k);
    uint8_t* ct = codes + ((long long)g * rows + (long long)rt * TILE) * pitch;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = r0 + 16 * i;
        const int s = block_scale<FMT>(quad_max(max_bits8(v[i])), up);
        const float inv = scale_inverse(s);
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] *= inv;
        const uint2 c = encode8<FMT>(v[i], s == 255);
        if (r < here) {
            if (FMT == OZK_MX_E2M1)
                *reinterpret_cast<uint32_t*>(ct + r * pitch + col / 2) = c.x;
            else
                *reinterpret_cast<uint2*>(ct + r * pitch + col) = c;
        }
        if ((lane16 & 3) == 0) sc[scale_slot(r, lane16 >> 2)] = (uint8_t)s;
    }
    __syncthreads();
    if (threadIdx.x < TILE_BYTES / 16)
        reinterpret_cast<uint4*>(scales + (long long)blockIdx.x * TILE_BYTES)[threadIdx.x] =
            reinterpret_cast<const uint4*>(sc)[threadIdx.x];
}

// ---- quantisation, any strides --------------------------------------------------------------------------------------
// The tile goes through shared memory as [element][row], so that whichever axis is contiguous is read along the lanes
// (`LOAD` 0: rows contiguous and 16-byte aligned, vector loads; 1: one element a lane along the rows; 2: along the
// contracted axis).  A thread then owns a block of a row pair (16-bit types: both rows' elements are one 32-bit word) or
// of one row (FP32), so a block's largest magnitude needs no exchange.  The codes go back through the same memory to
// leave as whole row segments.
template <typename T>
struct TileOf {
    static constexpr int PITCH = sizeof(T) == 4 ? 129 : 130;   // odd in 32-bit words: rows and columns free of conflicts
    static constexpr int BYTES = (TILE * PITCH * (int)sizeof(T) + 15) / 16 * 16;
};

template <typename T, int LOAD>
__device__ __forceinline__ void load_tile(T* __restrict__ tile, const T* __restrict__ xt, long long row_stride,
                                          long long k_stride, int here, int kept) {
    constexpr int P = TileOf<T>::PITCH;
    if (LOAD == 0) {
        constexpr int VEC = 16 / (int)sizeof(T);               // elements of a 16-byte load
        constexpr int PER = TILE / VEC;                        // loads of one k row of the tile
        constexpr int WORDS = (int)sizeof(T) * VEC / 4;
        static_assert(TILE * PER % THREADS == 0, "whole passes");
#pragma unroll 8
        for (int i = 0; i < TILE * PER / THREADS; i++) {
            const int id = threadIdx.x + i * THREADS;
            const int kk = id / PER, r = id % PER * VEC;
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (kk < kept) {
                const T* p = xt + kk * k_stride + r;
                if (r + VEC <= here) {
                    w = __ldg(reinterpret_cast<const uint4*>(p));
                } else {
                    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                        if (r + j < here) e[j] = p[j];
                }
            }
            uint32_t* d = reinterpret_cast<uint32_t*>(tile + kk * P + r);   // 4-byte aligned: P and r are even or T is
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};                    // 4 bytes wide
#pragma unroll
            for (int j = 0; j < WORDS; j++) d[j] = ww[j];
        }
    } else {
#pragma unroll 8
        for (int i = 0; i < TILE * TILE / THREADS; i++) {
            const int id = threadIdx.x + i * THREADS;
            const int kk = LOAD == 1 ? id / TILE : id % TILE, r = LOAD == 1 ? id % TILE : id / TILE;
            T e = from_f32<T>(0.0f);
            if (kk < kept && r < here) e = xt[r * row_stride + kk * k_stride];
            tile[kk * P + r] = e;
        }
    }
}

// The 32 values of block `b` of row `r` (FP32) or rows r, r + 1 (16-bit types) to codes and scale bytes
template <int FMT>
__device__ __forceinline__ void encode_block(const float* tile, int r, int b, bool up, uint4 (&c)[2], int& s) {
    constexpr int P = TileOf<float>::PITCH;
    const float* p = tile + b * BLOCK * P + r;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < BLOCK; j++) m = max(m, __float_as_uint(p[j * P]) & 0x7fffffffu);
    s = block_scale<FMT>(m, up);
    const float inv = scale_inverse(s);
    uint2 w[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = p[(8 * q + j) * P] * inv;
        w[q] = encode8<FMT>(v, s == 255);
    }
    c[0] = FMT == OZK_MX_E2M1 ? make_uint4(w[0].x, w[1].x, w[2].x, w[3].x) : make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
    c[1] = make_uint4(w[2].x, w[2].y, w[3].x, w[3].y);
}

__device__ __forceinline__ uint32_t bits_of_max(__half*, uint32_t m16) {
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m16)));
}
__device__ __forceinline__ uint32_t bits_of_max(__nv_bfloat16*, uint32_t m16) { return m16 << 16; }

template <typename T, int FMT>
__device__ __forceinline__ void encode_pair(const T* tile, int r, int b, bool up, uint4 (&c)[2][2], int (&s)[2]) {
    constexpr int P = TileOf<T>::PITCH;
    const T* p = tile + b * BLOCK * P + r;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < BLOCK; j++) m = __vmaxu2(m, *reinterpret_cast<const uint32_t*>(p + j * P) & 0x7fff7fffu);
#pragma unroll
    for (int h = 0; h < 2; h++) s[h] = block_scale<FMT>(bits_of_max((T*)nullptr, h ? m >> 16 : m & 0xffffu), up);
    const float inv[2] = {scale_inverse(s[0]), scale_inverse(s[1])};
    uint2 w[2][4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        float v[2][8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[0][j] = to_f32(p[(8 * q + j) * P]) * inv[0];
            v[1][j] = to_f32(p[(8 * q + j) * P + 1]) * inv[1];
        }
        w[0][q] = encode8<FMT>(v[0], s[0] == 255);
        w[1][q] = encode8<FMT>(v[1], s[1] == 255);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        c[h][0] = FMT == OZK_MX_E2M1 ? make_uint4(w[h][0].x, w[h][1].x, w[h][2].x, w[h][3].x)
                                     : make_uint4(w[h][0].x, w[h][0].y, w[h][1].x, w[h][1].y);
        c[h][1] = make_uint4(w[h][2].x, w[h][2].y, w[h][3].x, w[h][3].y);
    }
}

template <typename T, int FMT, int LOAD>
__global__ void __launch_bounds__(THREADS)
    quantize_tile_kernel(const T* __restrict__ x, long long group_stride, long long row_stride, long long k_stride,
                         int rows, int k, bool up, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(16) uint8_t sc[TILE_BYTES];
    constexpr int SEG = FMT == OZK_MX_E2M1 ? TILE / 2 : TILE;   // code bytes of a row of the tile
    constexpr int CP = SEG + 16;
    static_assert(TILE * CP <= TileOf<T>::BYTES, "codes fit where the values were");
    T* tile = reinterpret_cast<T*>(smem);
    const int ktiles = padded_k(k) / TILE, rtiles = row_tiles(rows);
    // rows contiguous: neighbouring CTAs take neighbouring row tiles, so that their reads share DRAM pages
    int kt, rt, g;
    if (LOAD == 2) {
        kt = (int)(blockIdx.x % (unsigned)ktiles);
        const int t = (int)(blockIdx.x / (unsigned)ktiles);
        rt = t % rtiles;
        g = t / rtiles;
    } else {
        rt = (int)(blockIdx.x % (unsigned)rtiles);
        const int t = (int)(blockIdx.x / (unsigned)rtiles);
        kt = t % ktiles;
        g = t / ktiles;
    }
    const int here = min(TILE, rows - rt * TILE), kept = min(TILE, k - kt * TILE);
    load_tile<T, LOAD>(tile, x + g * group_stride + (long long)rt * TILE * row_stride + (long long)kt * TILE * k_stride,
                       row_stride, k_stride, here, kept);
    __syncthreads();
    if constexpr (sizeof(T) == 4) {
        uint4 c[2][2];
        const int r = threadIdx.x & (TILE - 1);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            int s;
            const int b = (threadIdx.x >> 7) + 2 * i;
            encode_block<FMT>(tile, r, b, up, c[i], s);
            sc[scale_slot(r, b)] = (uint8_t)s;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; i++) {
            uint4* d = reinterpret_cast<uint4*>(smem + r * CP + ((threadIdx.x >> 7) + 2 * i) * (SEG / 4));
            d[0] = c[i][0];
            if (FMT != OZK_MX_E2M1) d[1] = c[i][1];
        }
    } else {
        uint4 c[2][2];
        int s[2];
        const int r = 2 * (threadIdx.x & 63), b = threadIdx.x >> 6;
        encode_pair<T, FMT>(tile, r, b, up, c, s);
        sc[scale_slot(r, b)] = (uint8_t)s[0];
        sc[scale_slot(r + 1, b)] = (uint8_t)s[1];
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint4* d = reinterpret_cast<uint4*>(smem + (r + h) * CP + b * (SEG / 4));
            d[0] = c[h][0];
            if (FMT != OZK_MX_E2M1) d[1] = c[h][1];
        }
    }
    __syncthreads();
    const long long pitch = code_pitch(FMT, k);
    uint8_t* ct = codes + ((long long)g * rows + (long long)rt * TILE) * pitch + (long long)kt * SEG;
    constexpr int VECS = SEG / 16;
#pragma unroll
    for (int i = 0; i < TILE * VECS / THREADS; i++) {
        const int id = threadIdx.x + i * THREADS;
        const int r = id / VECS, q = id % VECS;
        if (r < here)
            *reinterpret_cast<uint4*>(ct + r * pitch + 16 * q) = *reinterpret_cast<const uint4*>(smem + r * CP + 16 * q);
    }
    if (threadIdx.x < TILE_BYTES / 16)
        reinterpret_cast<uint4*>(scales + (((long long)g * rtiles + rt) * ktiles + kt) * TILE_BYTES)[threadIdx.x] =
            reinterpret_cast<const uint4*>(sc)[threadIdx.x];
}

// ---- the way back ---------------------------------------------------------------------------------------------------
// One CTA per scale tile, 16 lanes a row as in the quantisation; each value is one multiplication in FP32 and one
// rounding to the output type (none for the values of ordinary scales, which BF16 and FP32 hold exactly).
template <typename T, int FMT>
__global__ void __launch_bounds__(THREADS)
    dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int k,
                      T* __restrict__ out) {
    __shared__ __align__(16) uint8_t sc[TILE_BYTES];
    const int ktiles = padded_k(k) / TILE, rtiles = row_tiles(rows);
    const int kt = (int)(blockIdx.x % (unsigned)ktiles);
    const int t = (int)(blockIdx.x / (unsigned)ktiles);
    const int rt = t % rtiles, g = t / rtiles;
    const int lane16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int col = kt * TILE + lane16 * 8;
    const int here = min(TILE, rows - rt * TILE);
    const long long pitch = code_pitch(FMT, k);
    const uint8_t* ct = codes + ((long long)g * rows + (long long)rt * TILE) * pitch + (FMT == OZK_MX_E2M1 ? col / 2 : col);
    uint2 c[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = r0 + 16 * i;
        c[i] = make_uint2(0u, 0u);
        if (r < here) {
            if (FMT == OZK_MX_E2M1)
                c[i].x = __ldg(reinterpret_cast<const uint32_t*>(ct + r * pitch));
            else
                c[i] = __ldg(reinterpret_cast<const uint2*>(ct + r * pitch));
        }
    }
    if (threadIdx.x < TILE_BYTES / 16)
        reinterpret_cast<uint4*>(sc)[threadIdx.x] =
            __ldg(reinterpret_cast<const uint4*>(scales + (long long)blockIdx.x * TILE_BYTES) + threadIdx.x);
    __syncthreads();
    const bool whole = col + 8 <= k && (k * (int)sizeof(T)) % 16 == 0;
    const int count = max(0, k - col);
    T* ot = out + ((long long)g * rows + (long long)rt * TILE) * k + col;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = r0 + 16 * i;
        if (r >= here) continue;
        const float s = scale_value(sc[scale_slot(r, lane16 >> 2)]);
        float v[8];
        decode8<FMT>(c[i], v);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= s;
        store8(ot + (long long)r * k, whole, count, v);
    }
}

// ---- root-mean-square norm with an MX output -----------------------------------------------------------------------
// t = x (+ residual), y = t / sqrt(mean(t^2) + eps) weight, y quantised; t, rounded to the type of x, is the next
// residual.  Everything between the loads and the codes stays in FP32 registers: one pass over x and the residual, TPR
// threads a row with NC chunks of eight values each (longer rows read the rest a second time).  The sums are taken in a
// fixed order.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (TPR == 32) return v;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < TPR / 32 ? part[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T, typename W, int FMT, int TPR, int NC>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR)
    rms_norm_kernel(const T* __restrict__ x, long long x_stride, const T* __restrict__ residual, long long res_stride,
                    const W* __restrict__ weight, int rows, int d, float eps, bool aligned, bool up,
                    T* __restrict__ sum, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    __shared__ float part[32];
    constexpr int RPB = TPR == 32 ? 4 : 1;
    const long long row = (long long)blockIdx.x * RPB + (RPB == 1 ? 0 : threadIdx.x / TPR);
    const int t = RPB == 1 ? threadIdx.x : threadIdx.x % TPR;
    if (row >= rows) return;                                   // whole warps only (RPB > 1): no barrier follows them
    const int kp = padded_k(d), chunks = kp / 8;
    const T* xr = x + row * x_stride;
    const T* rr = residual ? residual + row * res_stride : nullptr;
    T* sr = sum ? sum + row * (long long)d : nullptr;

    float v[NC][8];
    float sq = 0.0f;
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
    auto note = [&](int c, const float (&o)[8]) {
        if (sr) store8(sr + c * 8, aligned && c * 8 + 8 <= d, max(0, d - c * 8), o);
#pragma unroll
        for (int j = 0; j < 8; j++) sq = fmaf(o[j], o[j], sq);
    };
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const int c = t + i * TPR;
        if (c < chunks) fetch(c, v[i]);
    }
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const int c = t + i * TPR;
        if (c < chunks) note(c, v[i]);
    }
    for (int c = t + NC * TPR; c < chunks; c += TPR) {
        float o[8];
        fetch(c, o);
        note(c, o);
    }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(sq, part) / (float)d + eps);

    const long long pitch = code_pitch(FMT, d);
    uint8_t* cr = codes + row * pitch;
    uint8_t* tr = scales + (row / TILE) * (long long)(kp / TILE) * TILE_BYTES + scale_slot((int)(row % TILE), 0);
    // 16 lanes hold a k tile of the row (chunks is a multiple of 16, so they are all in or all out)
    auto emit = [&](int c, float (&o)[8], bool in) {
        float w[8];
        load8(weight + c * 8, in && aligned && c * 8 + 8 <= d, in ? max(0, d - c * 8) : 0, w);
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = in ? o[j] * rstd * w[j] : 0.0f;
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
    };
#pragma unroll
    for (int i = 0; i < NC; i++) emit(t + i * TPR, v[i], t + i * TPR < chunks);
    for (int c0 = NC * TPR; c0 < chunks; c0 += TPR) {           // the same trips for every lane of a warp
        const int c = c0 + t;
        float o[8] = {};
        if (c < chunks) fetch(c, o);
        emit(c, o, c < chunks);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool fmt_ok(int fmt) { return fmt == OZK_MX_E2M1 || fmt == OZK_MX_E4M3; }

// CTAs of one scale tile each; -1 when they pass the grid's limit
long long tile_count(int groups, int rows, int k) {
    const long long n = (long long)groups * row_tiles(rows) * (padded_k(k) / TILE);
    return n <= 0x7fffffffLL ? n : -1;
}

template <typename T, int FMT>
int launch_quantize(const T* x, int groups, int rows, int k, long long gs, long long rs, long long ks, bool up,
                    uint8_t* codes, uint8_t* scales, cudaStream_t st) {
    const unsigned grid = (unsigned)tile_count(groups, rows, k);
    const long long size = (long long)sizeof(T);
    const bool base = aligned16(x) && (groups == 1 || gs * size % 16 == 0);
    if (ks == 1 && base && (rows == 1 || rs * size % 16 == 0)) {
        quantize_rows_kernel<T, FMT><<<grid, THREADS, 0, st>>>(x, gs, rs, rows, k, up, codes, scales);
    } else {
        constexpr int bytes = TileOf<T>::BYTES;
        const int load = rs == 1 && base && (k == 1 || ks * size % 16 == 0) ? 0 : rs == 1 || (rs < ks && ks != 1) ? 1 : 2;
        auto kern = load == 0 ? quantize_tile_kernel<T, FMT, 0>
                              : load == 1 ? quantize_tile_kernel<T, FMT, 1> : quantize_tile_kernel<T, FMT, 2>;
        if (bytes > 48 * 1024 - TILE_BYTES) {
            const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
            if (e != cudaSuccess) return OZK_ERR_CUDA_BASE + (int)e;
        }
        kern<<<grid, THREADS, bytes, st>>>(x, gs, rs, ks, rows, k, up, codes, scales);
    }
    OZK_CHECK_LAUNCH();
    return OZK_OK;
}

template <typename T>
int launch_dequantize(const uint8_t* codes, const uint8_t* scales, int fmt, int groups, int rows, int k, T* out,
                      cudaStream_t st) {
    const unsigned grid = (unsigned)tile_count(groups, rows, k);
    if (fmt == OZK_MX_E2M1)
        dequantize_kernel<T, OZK_MX_E2M1><<<grid, THREADS, 0, st>>>(codes, scales, rows, k, out);
    else
        dequantize_kernel<T, OZK_MX_E4M3><<<grid, THREADS, 0, st>>>(codes, scales, rows, k, out);
    OZK_CHECK_LAUNCH();
    return OZK_OK;
}

struct NormArgs {
    const void *x, *residual, *weight;
    long long x_stride, res_stride;
    int rows, d;
    float eps;
    bool up;
    void* sum;
    uint8_t *codes, *scales;
    cudaStream_t st;
};

template <typename T, typename W, int FMT>
int launch_norm(const NormArgs& a) {
    const long long size = (long long)sizeof(T);
    const bool aligned = aligned16(a.x) && aligned16(a.residual) && aligned16(a.weight) && aligned16(a.sum) &&
                         (a.rows == 1 || (a.x_stride * size % 16 == 0 && (!a.residual || a.res_stride * size % 16 == 0) &&
                                          (!a.sum || a.d * size % 16 == 0)));
    // threads a row: enough that a row's values stay in registers (4 chunks of eight a thread), a warp for short rows
    const int d = a.d;
#define OZK_NORM(TPR, NC)                                                                                            \
    rms_norm_kernel<T, W, FMT, TPR, NC>                                                                              \
        <<<(unsigned)((a.rows + (TPR == 32 ? 3 : 0)) / (TPR == 32 ? 4 : 1)), TPR == 32 ? 128 : TPR, 0, a.st>>>(      \
            static_cast<const T*>(a.x), a.x_stride, static_cast<const T*>(a.residual), a.res_stride,                 \
            static_cast<const W*>(a.weight), a.rows, d, a.eps, aligned, a.up, static_cast<T*>(a.sum), a.codes, a.scales)
    if (d <= 1024) OZK_NORM(32, 4);
    else if (d <= 4096) OZK_NORM(256, 2);
    else if (d <= 8192) OZK_NORM(256, 4);
    else OZK_NORM(1024, 4);
#undef OZK_NORM
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

extern "C" size_t ozk_mx_code_bytes(int fmt, int groups, int rows, int k) {
    if (!fmt_ok(fmt) || groups < 1 || rows < 1 || k < 1 || k > OZK_MX_KMAX) return 0;
    return (size_t)groups * rows * code_pitch(fmt, k);
}

extern "C" size_t ozk_mx_scale_bytes(int groups, int rows, int k) {
    if (groups < 1 || rows < 1 || k < 1 || k > OZK_MX_KMAX) return 0;
    return (size_t)groups * scale_group_bytes(rows, k);
}

extern "C" int ozk_mx_quantize(const void* x, int dtype, int groups, int rows, int k, int64_t group_stride,
                               int64_t row_stride, int64_t k_stride, int fmt, int round_up, uint8_t* codes,
                               uint8_t* scales, ozk_stream_t stream) {
    if (!x || !codes || !scales || !fmt_ok(fmt) || groups < 1 || rows < 1 || k < 1 || k > OZK_MX_KMAX) return OZK_ERR_ARG;
    if (group_stride < 0 || row_stride < 0 || k_stride < 0 || !aligned16(codes) || !aligned16(scales)) return OZK_ERR_ARG;
    if (tile_count(groups, rows, k) < 0) return OZK_ERR_ARG;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define OZK_QUANT(T)                                                                                                 \
    (fmt == OZK_MX_E2M1                                                                                              \
         ? launch_quantize<T, OZK_MX_E2M1>(static_cast<const T*>(x), groups, rows, k, group_stride, row_stride,      \
                                           k_stride, round_up != 0, codes, scales, st)                               \
         : launch_quantize<T, OZK_MX_E4M3>(static_cast<const T*>(x), groups, rows, k, group_stride, row_stride,      \
                                           k_stride, round_up != 0, codes, scales, st))
    switch (dtype) {
        case OZK_F32: return OZK_QUANT(float);
        case OZK_F16: return OZK_QUANT(__half);
        case OZK_BF16: return OZK_QUANT(__nv_bfloat16);
        default: return OZK_ERR_ARG;
    }
#undef OZK_QUANT
}

extern "C" int ozk_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int fmt, int groups, int rows, int k,
                                 void* out, int dtype, ozk_stream_t stream) {
    if (!codes || !scales || !out || !fmt_ok(fmt) || groups < 1 || rows < 1 || k < 1 || k > OZK_MX_KMAX)
        return OZK_ERR_ARG;
    if (!aligned16(codes) || !aligned16(scales) || !aligned16(out) || tile_count(groups, rows, k) < 0) return OZK_ERR_ARG;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (dtype) {
        case OZK_F32: return launch_dequantize(codes, scales, fmt, groups, rows, k, static_cast<float*>(out), st);
        case OZK_F16: return launch_dequantize(codes, scales, fmt, groups, rows, k, static_cast<__half*>(out), st);
        case OZK_BF16:
            return launch_dequantize(codes, scales, fmt, groups, rows, k, static_cast<__nv_bfloat16*>(out), st);
        default: return OZK_ERR_ARG;
    }
}

extern "C" int ozk_mx_rms_norm(const void* x, const void* residual, const void* weight, int dtype, int weight_f32,
                               int rows, int d, int64_t x_stride, int64_t residual_stride, float eps, int fmt,
                               int round_up, void* sum, uint8_t* codes, uint8_t* scales, ozk_stream_t stream) {
    if (!x || !weight || !codes || !scales || !fmt_ok(fmt) || rows < 1 || d < 1 || d > OZK_MX_KMAX) return OZK_ERR_ARG;
    if (!(eps > 0.0f) || !(eps < INFINITY) || x_stride < 0 || residual_stride < 0) return OZK_ERR_ARG;
    if (!aligned16(codes) || !aligned16(scales)) return OZK_ERR_ARG;
    const NormArgs a = {x,    residual,      weight, x_stride, residual_stride, rows,
                        d,    eps,           round_up != 0,    sum,  codes,  scales,
                        reinterpret_cast<cudaStream_t>(stream)};
    switch (dtype) {
        case OZK_F32: return dispatch_norm<float>(a, true, fmt);
        case OZK_F16: return dispatch_norm<__half>(a, weight_f32 != 0, fmt);
        case OZK_BF16: return dispatch_norm<__nv_bfloat16>(a, weight_f32 != 0, fmt);
        default: return OZK_ERR_ARG;
    }
}
