// Operand preparation for the microscaled products: quantisation to MX codes and scales and the way back; and the linear
// layer's two passes, which are quantisations and products in a row.
#include "mx_common.cuh"

using namespace ozk_mx;

namespace {

constexpr int THREADS = 256;

// ---- quantisation ---------------------------------------------------------------------------------------------------
// A job reads an I x J matrix (times groups; element (i, j) at x + i si + j sj) in tiles of 128 x 128 and writes it as the
// operand that contracts j (vectors are rows, `row_*`), as the one that contracts i (vectors are columns, `col_*`), or
// as both from one read.
struct QuantJob {
    const void* x;
    long long gs, si, sj;
    int groups, I, J;
    uint8_t *row_codes, *row_scales, *col_codes, *col_scales;
    uintptr_t begin, end;                    // the bytes between its first and last element
};

__device__ __forceinline__ void copy_scale_tile(uint8_t* __restrict__ to, const uint8_t* sc) {
    if (threadIdx.x < TILE_BYTES / 16)
        reinterpret_cast<uint4*>(to)[threadIdx.x] = reinterpret_cast<const uint4*>(sc)[threadIdx.x];
}

// Eight consecutive FP32 values that need not be aligned to 16 bytes: the three aligned vectors around them, shifted into
// place, where those lie within [begin, end); one by one otherwise.
__device__ __forceinline__ void load8_any(const float* __restrict__ p, int count, uintptr_t begin, uintptr_t end,
                                          float (&v)[8]) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), a0 = at & ~(uintptr_t)15;
    const uint32_t sh = (uint32_t)(at & 15);
    if (count < 8 || a0 < begin || a0 + 48 > end) {
        load8(p, false, count, v);
        return;
    }
    float w[14];
#pragma unroll
    for (int q = 0; q < 3; q++) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(a0) + q);
        w[4 * q] = u.x; w[4 * q + 1] = u.y; w[4 * q + 2] = u.z; w[4 * q + 3] = u.w;
    }
    w[12] = w[13] = 0.0f;
    if (sh & 8u) {
#pragma unroll
        for (int j = 0; j < 12; j++) w[j] = w[j + 2];
    }
    if (sh & 4u) {
#pragma unroll
        for (int j = 0; j < 12; j++) w[j] = w[j + 1];
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = w[j];
}

// One row's eight values per lane (16 lanes a row of the tile) to codes in global memory and the scale byte in `sc`: a
// block of 32 is four lanes, its largest magnitude two shuffles away.
template <int FMT>
__device__ __forceinline__ void emit_row(float (&v)[8], uint32_t max_bits, bool up, int r, int here, int lane16,
                                         uint8_t* __restrict__ ct, long long pitch, uint8_t* sc) {
    const int s = block_scale<FMT>(quad_max(max_bits), up);
    const float inv = scale_inverse(s);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] *= inv;
    const uint2 c = encode8<FMT>(v, s == 255);
    if (r < here) {
        if (FMT == OZK_MX_E2M1)
            *reinterpret_cast<uint32_t*>(ct + r * pitch + lane16 * 4) = c.x;
        else
            *reinterpret_cast<uint2*>(ct + r * pitch + lane16 * 8) = c;
    }
    if ((lane16 & 3) == 0) sc[scale_slot(r, lane16 >> 2)] = (uint8_t)s;
}

// The same for eight 16-bit values as they lie in memory (aligned; the first `count` of them, zeros behind)
template <typename T>
__device__ __forceinline__ uint4 load8_raw(const T* __restrict__ p, int count) {
    if (count >= 8) return __ldg(reinterpret_cast<const uint4*>(p));
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (count > 0) {
        uint16_t e[8] = {};
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < count) e[j] = reinterpret_cast<const uint16_t*>(p)[j];
        w = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                       e[6] | (uint32_t)e[7] << 16);
    }
    return w;
}

// A thread's eight rows (r0 + 16 i) of a tile of 16-bit values, eight values each from column col0 + 8 lane16 of rows that
// have J; `first` is column 0 of the tile's first row, of `rows`; zeros outside
template <typename T, bool ALIGNED>
__device__ __forceinline__ void load_rows_raw(const QuantJob& q, const T* __restrict__ first, int rows, int col0, int r0,
                                              int lane16, uint4 (&raw)[8]) {
    const long long row_stride = q.si;
    const int J = q.J;
    const int col = col0 + lane16 * 8;
    if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            raw[i] = load8_raw(first + (long long)(r0 + 16 * i) * row_stride + col, r0 + 16 * i < rows ? J - col : 0);
    } else {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
            uint4 tail[4];                                      // the granule behind a row's last lane
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = r0 + 16 * (h + i);
                const uintptr_t row = reinterpret_cast<uintptr_t>(first + (long long)r * row_stride);
                const uintptr_t end = r < rows ? row + 2 * (uintptr_t)J : 0;
                const uintptr_t at = (row & ~(uintptr_t)15) + 2 * (uintptr_t)col;
                raw[h + i] = load_granule(at, end, q.begin, q.end);
                tail[i] = make_uint4(0u, 0u, 0u, 0u);
                if (lane16 == 15) tail[i] = load_granule(at + 16, end, q.begin, q.end);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t sh = (uint32_t)(reinterpret_cast<uintptr_t>(first + (long long)(r0 + 16 * (h + i)) * row_stride) & 15);
                const uint4 n = next_lane(raw[h + i]);
                raw[h + i] = keep8(shift_granules(raw[h + i], lane16 == 15 ? tail[i] : n, sh), J - col);
            }
        }
    }
}

template <typename T, int FMT>
__device__ __forceinline__ void emit_raw(uint4 raw, bool up, int r, int here, int lane16, uint8_t* __restrict__ ct,
                                         long long pitch, uint8_t* sc) {
    const T* const type = nullptr;
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    const float2 m = unpack2(__vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu),
                                      __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu)), type);
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 f = unpack2(w[j], type);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
    }
    emit_row<FMT>(v, max(__float_as_uint(m.x), __float_as_uint(m.y)), up, r, here, lane16, ct, pitch, sc);
}

// The row operand, rows contiguous.  One CTA per scale tile; a thread's loads are issued before the first is used, and the
// tile's 512 scale bytes leave as one contiguous store.  ALIGNED: rows start on 16-byte boundaries.  bf16 16384 x 8192 to
// e4m3: 66 us, 6.1 TB/s, issue slots 71 % (104 us with the values unpacked to FP32 on arrival, three CTAs an SM instead of
// four); 8192 x 4097: 36 us, 2.9 TB/s.  FP32 8192 x 8192: 52 us, 6.5 TB/s; 8192 x 4097: 49 us, 3.5 TB/s.
template <typename T, int FMT, bool ALIGNED>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 && ALIGNED ? 4 : 3)
    quantize_rows_kernel(const __grid_constant__ QuantJob q, bool up) {
    __shared__ __align__(16) uint8_t sc[TILE_BYTES];
    const int ktiles = padded_k(q.J) / TILE, rtiles = row_tiles(q.I);
    const int kt = (int)(blockIdx.x % (unsigned)ktiles);
    const int t = (int)(blockIdx.x / (unsigned)ktiles);
    const int rt = t % rtiles, g = t / rtiles;
    const int lane16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int col = kt * TILE + lane16 * 8;
    const int here = min(TILE, q.I - rt * TILE);
    const T* xt = static_cast<const T*>(q.x) + g * q.gs + (long long)rt * TILE * q.si + col;
    const int count = max(0, q.J - col);

    const long long pitch = code_pitch(FMT, q.J);
    uint8_t* ct = q.row_codes + ((long long)g * q.I + (long long)rt * TILE) * pitch + kt * (FMT == OZK_MX_E2M1 ? 64 : 128);
    if constexpr (sizeof(T) == 2) {
        // the words as they are until they are encoded: half the registers, and magnitudes ordered like their bits
        uint4 raw[8];
        load_rows_raw<T, ALIGNED>(q, xt - col, here, kt * TILE, r0, lane16, raw);
#pragma unroll
        for (int i = 0; i < 8; i++) emit_raw<T, FMT>(raw[i], up, r0 + 16 * i, here, lane16, ct, pitch, sc);
    } else {
        float v[8][8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = r0 + 16 * i;
            const int n = r < here ? count : 0;
            if (ALIGNED) load8(xt + (long long)r * q.si, n >= 8, n, v[i]);
            else load8_any(xt + (long long)r * q.si, n, q.begin, q.end, v[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) emit_row<FMT>(v[i], max_bits8(v[i]), up, r0 + 16 * i, here, lane16, ct, pitch, sc);
    }
    __syncthreads();
    copy_scale_tile(q.row_scales + (long long)blockIdx.x * TILE_BYTES, sc);
}

// The 32 values of one block, largest magnitude `m` (FP32 bits), to its code bytes
template <int FMT, typename Get>
__device__ __forceinline__ int encode_block(uint32_t m, bool up, uint4 (&c)[2], Get get) {
    const int s = block_scale<FMT>(m, up);
    const float inv = scale_inverse(s);
    uint2 w[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = get(8 * q + j) * inv;
        w[q] = encode8<FMT>(v, s == 255);
    }
    c[0] = FMT == OZK_MX_E2M1 ? make_uint4(w[0].x, w[1].x, w[2].x, w[3].x) : make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
    c[1] = make_uint4(w[2].x, w[2].y, w[3].x, w[3].y);
    return s;
}

// The column operand, or (FP32, rows aligned) both operands, of one or two jobs in one launch; any strides.  A thread owns
// a block of 32 values down a column (FP32) or a pair of columns (16-bit types), which it reads straight into registers: a
// warp reads a row's neighbouring values, nothing is transposed in memory, and a block's largest magnitude needs no
// exchange.  Only the codes go through shared memory, to leave as whole segments of the operand's vectors.  The row operand
// reads the tile again.  FP32 5001 x 4095 down the columns to e2m1: 18 us, 5.1 TB/s.
template <typename T, int FMT>
__global__ void __launch_bounds__(THREADS)
    quantize_dual_kernel(const __grid_constant__ QuantJob q0, const __grid_constant__ QuantJob q1, unsigned tiles0, bool up) {
    constexpr int SEG = FMT == OZK_MX_E2M1 ? TILE / 2 : TILE;   // code bytes of a vector of the tile
    constexpr int CP = SEG + 16;
    __shared__ __align__(16) uint8_t staged[TILE * CP];
    __shared__ __align__(16) uint8_t sc[2][TILE_BYTES];
    const bool second = blockIdx.x >= tiles0;
    const QuantJob& q = second ? q1 : q0;
    const unsigned tile = second ? blockIdx.x - tiles0 : blockIdx.x;
    const int jtiles = padded_k(q.J) / TILE, itiles = padded_k(q.I) / TILE;
    const int jt = (int)(tile % (unsigned)jtiles);
    const int t = (int)(tile / (unsigned)jtiles);
    const int it = t % itiles, g = t / itiles;
    const int rows = min(TILE, q.I - it * TILE), cols = min(TILE, q.J - jt * TILE);
    const T* xt = static_cast<const T*>(q.x) + g * q.gs + (long long)it * TILE * q.si + (long long)jt * TILE * q.sj;

    if (q.col_codes) {
        if constexpr (sizeof(T) == 4) {
            const int c = threadIdx.x & (TILE - 1);
#pragma unroll 1
            for (int h = 0; h < 2; h++) {
                const int b = (threadIdx.x >> 7) + 2 * h;
                float v[BLOCK];
                float m = 0.0f;
                const T* p = xt + (long long)(b * BLOCK) * q.si + c * q.sj;
#pragma unroll
                for (int j = 0; j < BLOCK; j++) v[j] = (c < cols && b * BLOCK + j < rows) ? __ldg(p + j * q.si) : 0.0f;
#pragma unroll
                for (int j = 0; j < BLOCK; j++) m = max_magnitude(m, v[j]);
                uint4 o[2];
                sc[0][scale_slot(c, b)] = (uint8_t)encode_block<FMT>(__float_as_uint(m), up, o, [&](int j) { return v[j]; });
                uint4* d = reinterpret_cast<uint4*>(staged + c * CP + b * (SEG / 4));
                d[0] = o[0];
                if (FMT != OZK_MX_E2M1) d[1] = o[1];
            }
        } else {
            const int c = 2 * (threadIdx.x & 63), b = threadIdx.x >> 6;
            uint32_t v[BLOCK];
            const T* p = xt + (long long)(b * BLOCK) * q.si + c * q.sj;
#pragma unroll
            for (int j = 0; j < BLOCK; j++) {
                v[j] = 0u;
                if (b * BLOCK + j < rows) {
                    if (c < cols) v[j] = __ldg(reinterpret_cast<const unsigned short*>(p + j * q.si));
                    if (c + 1 < cols) v[j] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(p + j * q.si + q.sj)) << 16;
                }
            }
            uint32_t m = 0;                                      // magnitudes of 16-bit types are ordered like their bits
#pragma unroll
            for (int j = 0; j < BLOCK; j++) m = __vmaxu2(m, v[j] & 0x7fff7fffu);
            const T* const type = nullptr;
            uint4 o[2];
            uint4* d = reinterpret_cast<uint4*>(staged + c * CP + b * (SEG / 4));
            sc[0][scale_slot(c, b)] = (uint8_t)encode_block<FMT>(__float_as_uint(unpack2(m, type).x), up, o,
                                                                 [&](int j) { return unpack2(v[j], type).x; });
            d[0] = o[0];
            if (FMT != OZK_MX_E2M1) d[1] = o[1];
            d = reinterpret_cast<uint4*>(staged + (c + 1) * CP + b * (SEG / 4));
            sc[0][scale_slot(c + 1, b)] = (uint8_t)encode_block<FMT>(__float_as_uint(unpack2(m, type).y), up, o,
                                                                     [&](int j) { return unpack2(v[j], type).y; });
            d[0] = o[0];
            if (FMT != OZK_MX_E2M1) d[1] = o[1];
        }
    }
    if (sizeof(T) == 4 && q.row_codes) {
        const int lane16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
        const long long pitch = code_pitch(FMT, q.J);
        uint8_t* ct = q.row_codes + ((long long)g * q.I + (long long)it * TILE) * pitch + (long long)jt * SEG;
        const int count = max(0, cols - lane16 * 8);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float v[4][8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = r0 + 16 * (4 * h + i), n = r < rows ? count : 0;
                load8(xt + (long long)r * q.si + lane16 * 8, n >= 8, n, v[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) emit_row<FMT>(v[i], max_bits8(v[i]), up, r0 + 16 * (4 * h + i), rows, lane16, ct, pitch, sc[1]);
        }
    }
    __syncthreads();
    if (q.col_codes) {
        const long long pitch = code_pitch(FMT, q.I);
        uint8_t* ct = q.col_codes + ((long long)g * q.J + (long long)jt * TILE) * pitch + (long long)it * SEG;
        constexpr int VECS = SEG / 16;
#pragma unroll
        for (int i = 0; i < TILE * VECS / THREADS; i++) {
            const int id = threadIdx.x + i * THREADS;
            const int r = id / VECS, k = id % VECS;
            if (r < cols)
                *reinterpret_cast<uint4*>(ct + r * pitch + 16 * k) = *reinterpret_cast<const uint4*>(staged + r * CP + 16 * k);
        }
        copy_scale_tile(q.col_scales + (((long long)g * jtiles + jt) * itiles + it) * TILE_BYTES, sc[0]);
    }
    if (sizeof(T) == 4 && q.row_codes)
        copy_scale_tile(q.row_scales + (((long long)g * itiles + it) * jtiles + jt) * TILE_BYTES, sc[1]);
}

// Column operands, both operands, or several jobs, of 16-bit matrices with contiguous rows, from one read: 16 lanes load a
// row's 128 values, the row operand is encoded from those registers, and the tile goes to shared memory (rows 16 bytes
// apart from a multiple of 128: neither its rows nor its columns meet in a bank), from which the column operand is encoded
// as above.  bf16 16384 x 8192 to e4m3: columns 69 us, 5.9 TB/s (83 us straight from global memory), both 103 us, 5.3 TB/s
// (134 us when the tile was read from global memory twice).
template <typename T, int FMT, bool ALIGNED>
__global__ void __launch_bounds__(THREADS, ALIGNED ? 4 : 3)
    quantize_shared_kernel(const __grid_constant__ QuantJob q0, const __grid_constant__ QuantJob q1, unsigned tiles0, bool up) {
    constexpr int SEG = FMT == OZK_MX_E2M1 ? TILE / 2 : TILE, CP = SEG + 16, PITCH = TILE * 2 + 16;
    __shared__ __align__(16) uint8_t tile_mem[TILE * PITCH];
    __shared__ __align__(16) uint8_t sc[2][TILE_BYTES];
    static_assert(TILE * CP <= TILE * PITCH, "codes fit where the values were");
    const bool second = blockIdx.x >= tiles0;
    const QuantJob& q = second ? q1 : q0;
    const unsigned tile = second ? blockIdx.x - tiles0 : blockIdx.x;
    const int jtiles = padded_k(q.J) / TILE, itiles = padded_k(q.I) / TILE;
    const int jt = (int)(tile % (unsigned)jtiles);
    const int t = (int)(tile / (unsigned)jtiles);
    const int it = t % itiles, g = t / itiles;
    const int rows = min(TILE, q.I - it * TILE), cols = min(TILE, q.J - jt * TILE);
    const int lane16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const T* xt = static_cast<const T*>(q.x) + g * q.gs + (long long)it * TILE * q.si + (long long)jt * TILE;
    const T* const type = nullptr;

    uint4 raw[8];
    load_rows_raw<T, ALIGNED>(q, xt - jt * TILE, rows, jt * TILE, r0, lane16, raw);
    if (q.col_codes) {
#pragma unroll
        for (int i = 0; i < 8; i++) *reinterpret_cast<uint4*>(tile_mem + (r0 + 16 * i) * PITCH + lane16 * 16) = raw[i];
    }
    if (q.row_codes) {
        const long long pitch = code_pitch(FMT, q.J);
        uint8_t* ct = q.row_codes + ((long long)g * q.I + (long long)it * TILE) * pitch + (long long)jt * SEG;
#pragma unroll
        for (int i = 0; i < 8; i++) emit_raw<T, FMT>(raw[i], up, r0 + 16 * i, rows, lane16, ct, pitch, sc[1]);
    }
    __syncthreads();
    if (q.col_codes) {
        const int c = 2 * (threadIdx.x & 63), b = threadIdx.x >> 6;
        uint32_t v[BLOCK], m = 0;
#pragma unroll
        for (int j = 0; j < BLOCK; j++) v[j] = *reinterpret_cast<const uint32_t*>(tile_mem + (b * BLOCK + j) * PITCH + c * 2);
#pragma unroll
        for (int j = 0; j < BLOCK; j++) m = __vmaxu2(m, v[j] & 0x7fff7fffu);
        __syncthreads();                                        // all values are in registers: the codes take their place
        uint4 o[2];
        uint4* d = reinterpret_cast<uint4*>(tile_mem + c * CP + b * (SEG / 4));
        sc[0][scale_slot(c, b)] = (uint8_t)encode_block<FMT>(__float_as_uint(unpack2(m, type).x), up, o,
                                                             [&](int j) { return unpack2(v[j], type).x; });
        d[0] = o[0];
        if (FMT != OZK_MX_E2M1) d[1] = o[1];
        d = reinterpret_cast<uint4*>(tile_mem + (c + 1) * CP + b * (SEG / 4));
        sc[0][scale_slot(c + 1, b)] = (uint8_t)encode_block<FMT>(__float_as_uint(unpack2(m, type).y), up, o,
                                                                 [&](int j) { return unpack2(v[j], type).y; });
        d[0] = o[0];
        if (FMT != OZK_MX_E2M1) d[1] = o[1];
        __syncthreads();
        const long long pitch = code_pitch(FMT, q.I);
        uint8_t* ct = q.col_codes + ((long long)g * q.J + (long long)jt * TILE) * pitch + (long long)it * SEG;
        constexpr int VECS = SEG / 16;
#pragma unroll
        for (int i = 0; i < TILE * VECS / THREADS; i++) {
            const int id = threadIdx.x + i * THREADS;
            const int r = id / VECS, k = id % VECS;
            if (r < cols)
                *reinterpret_cast<uint4*>(ct + r * pitch + 16 * k) = *reinterpret_cast<const uint4*>(tile_mem + r * CP + 16 * k);
        }
        copy_scale_tile(q.col_scales + (((long long)g * jtiles + jt) * itiles + it) * TILE_BYTES, sc[0]);
    }
    if (q.row_codes)
        copy_scale_tile(q.row_scales + (((long long)g * itiles + it) * jtiles + jt) * TILE_BYTES, sc[1]);
}

// ---- the way back ---------------------------------------------------------------------------------------------------
// One CTA per scale tile, 16 lanes a row as in the quantisation; each value is one multiplication in FP32 and one
// rounding to the output type (none for the values of ordinary scales, which BF16 and FP32 hold exactly).  e4m3
// 16384 x 8192 to bf16: 63 us, 6.4 TB/s.
template <typename T, int FMT, bool ALIGNED>
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
    T* ot = out + ((long long)g * rows + (long long)rt * TILE) * k + kt * TILE;
    auto values = [&](int i, float (&v)[8]) {
        const float s = scale_value(sc[scale_slot(r0 + 16 * i, lane16 >> 2)]);
        decode8<FMT>(c[i], v);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= s;
    };
    if (ALIGNED) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = r0 + 16 * i;
            if (r >= here) continue;
            float v[8];
            values(i, v);
            store8(ot + (long long)r * k + lane16 * 8, col + 8 <= k, max(0, k - col), v);
        }
    } else {
        // rows that start anywhere: through shared memory, so that a warp's lanes write neighbouring elements
        extern __shared__ __align__(16) uint8_t smem[];
        T* tile = reinterpret_cast<T*>(smem);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float v[8];
            values(i, v);
            store8(tile + (r0 + 16 * i) * TILE + lane16 * 8, true, 8, v);
        }
        __syncthreads();
        const int cols = min(TILE, k - kt * TILE);
        for (int r = threadIdx.x >> 5; r < here; r += THREADS / 32)
#pragma unroll
            for (int j = 0; j < TILE / 32; j++) {
                const int e = (threadIdx.x & 31) + 32 * j;
                if (e < cols) ot[(long long)r * k + e] = tile[r * TILE + e];
            }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
// CTAs of one scale tile each; -1 when they pass the grid's limit
long long tile_count(int groups, int rows, int k) {
    const long long n = (long long)groups * row_tiles(rows) * (padded_k(k) / TILE);
    return n <= 0x7fffffffLL ? n : -1;
}

template <typename T, int FMT>
int launch_rows(const QuantJob& q, bool aligned, bool up, cudaStream_t st) {
    const unsigned grid = (unsigned)tile_count(q.groups, q.I, q.J);
    if (aligned) quantize_rows_kernel<T, FMT, true><<<grid, THREADS, 0, st>>>(q, up);
    else quantize_rows_kernel<T, FMT, false><<<grid, THREADS, 0, st>>>(q, up);
    OZK_CHECK_LAUNCH();
    return OZK_OK;
}

template <typename T, int FMT>
int launch_dual(const QuantJob& a, const QuantJob& b, bool up, cudaStream_t st) {
    const unsigned t0 = (unsigned)tile_count(a.groups, a.I, a.J);
    const unsigned t1 = b.x ? (unsigned)tile_count(b.groups, b.I, b.J) : 0u;
    quantize_dual_kernel<T, FMT><<<t0 + t1, THREADS, 0, st>>>(a, b, t0, up);
    OZK_CHECK_LAUNCH();
    return OZK_OK;
}

// `unit` bytes divide the starts of all rows (along i) of the job
bool rows_aligned(const QuantJob& q, long long size, uintptr_t unit) {
    return q.sj == 1 && reinterpret_cast<uintptr_t>(q.x) % unit == 0 && (q.I == 1 || q.si * size % (long long)unit == 0) &&
           (q.groups == 1 || q.gs * size % (long long)unit == 0);
}

template <typename T, int FMT>
int launch_shared(const QuantJob& a, const QuantJob& b, bool up, cudaStream_t st) {
    const unsigned t0 = (unsigned)tile_count(a.groups, a.I, a.J);
    const unsigned t1 = b.x ? (unsigned)tile_count(b.groups, b.I, b.J) : 0u;
    if (rows_aligned(a, 2, 16) && (!b.x || rows_aligned(b, 2, 16)))
        quantize_shared_kernel<T, FMT, true><<<t0 + t1, THREADS, 0, st>>>(a, b, t0, up);
    else
        quantize_shared_kernel<T, FMT, false><<<t0 + t1, THREADS, 0, st>>>(a, b, t0, up);
    OZK_CHECK_LAUNCH();
    return OZK_OK;
}

QuantJob swapped(const QuantJob& q) {
    QuantJob t = q;
    t.si = q.sj; t.sj = q.si; t.I = q.J; t.J = q.I;
    t.row_codes = q.col_codes; t.row_scales = q.col_scales; t.col_codes = q.row_codes; t.col_scales = q.row_scales;
    return t;
}

// One direction of a job (the row operand of q): the rows kernel where the contracted axis is contiguous, the column
// operand of the matrix read the other way otherwise
template <typename T, int FMT>
int quantize_one(QuantJob q, bool up, cudaStream_t st) {
    const long long size = (long long)sizeof(T);
    q.col_codes = q.col_scales = nullptr;
    if (q.sj == 1) {
        return launch_rows<T, FMT>(q, rows_aligned(q, size, 16), up, st);
    }
    const QuantJob t = swapped(q);
    if constexpr (sizeof(T) == 2)
        if (t.sj == 1) return launch_shared<T, FMT>(t, QuantJob{}, up, st);
    return launch_dual<T, FMT>(t, QuantJob{}, up, st);
}

// Jobs of one type: in one launch where a row operand has to be written beside a column operand or there are two jobs,
// and the alignment allows; one launch per operand otherwise
template <typename T, int FMT>
int quantize_jobs(const QuantJob* jobs, int count, bool up, cudaStream_t st) {
    bool joint = true;
    for (int i = 0; i < count; i++) {
        const bool both = jobs[i].row_codes && jobs[i].col_codes;
        // (FP32 rows that are not aligned are read by the rows kernel, whose loads are vectors all the same)
        if (sizeof(T) == 2 ? jobs[i].sj != 1 : !rows_aligned(jobs[i], 4, 16)) joint = false;
        if (count == 1 && !both) joint = false;
    }
    long long tiles = 0;
    for (int i = 0; i < count; i++) tiles += tile_count(jobs[i].groups, jobs[i].I, jobs[i].J);
    if (joint && tiles <= 0x7fffffffLL) {
        const QuantJob second = count > 1 ? jobs[1] : QuantJob{};
        if constexpr (sizeof(T) == 2) return launch_shared<T, FMT>(jobs[0], second, up, st);
        else return launch_dual<T, FMT>(jobs[0], second, up, st);
    }
    for (int i = 0; i < count; i++) {
        int rc = OZK_OK;
        if (jobs[i].row_codes) rc = quantize_one<T, FMT>(jobs[i], up, st);
        if (rc == OZK_OK && jobs[i].col_codes) rc = quantize_one<T, FMT>(swapped(jobs[i]), up, st);
        if (rc != OZK_OK) return rc;
    }
    return OZK_OK;
}

int quantize(QuantJob* jobs, int count, int dtype, int fmt, bool up, cudaStream_t st) {
    for (int i = 0; i < count; i++) {
        QuantJob& q = jobs[i];
        const long long last = (q.groups - 1) * q.gs + (q.I - 1) * q.si + (q.J - 1) * q.sj;
        q.begin = reinterpret_cast<uintptr_t>(q.x);
        q.end = q.begin + (uintptr_t)(last + 1) * (dtype == OZK_F32 ? 4 : 2);
    }
    switch (dtype) {
        case OZK_F32:
            return fmt == OZK_MX_E2M1 ? quantize_jobs<float, OZK_MX_E2M1>(jobs, count, up, st)
                                      : quantize_jobs<float, OZK_MX_E4M3>(jobs, count, up, st);
        case OZK_F16:
            return fmt == OZK_MX_E2M1 ? quantize_jobs<__half, OZK_MX_E2M1>(jobs, count, up, st)
                                      : quantize_jobs<__half, OZK_MX_E4M3>(jobs, count, up, st);
        case OZK_BF16:
            return fmt == OZK_MX_E2M1 ? quantize_jobs<__nv_bfloat16, OZK_MX_E2M1>(jobs, count, up, st)
                                      : quantize_jobs<__nv_bfloat16, OZK_MX_E4M3>(jobs, count, up, st);
        default: return OZK_ERR_ARG;
    }
}

template <typename T, int FMT>
int launch_dequantize_fmt(const uint8_t* codes, const uint8_t* scales, int groups, int rows, int k, T* out, cudaStream_t st) {
    const unsigned grid = (unsigned)tile_count(groups, rows, k);
    if ((long long)k * (int)sizeof(T) % 16 == 0 || (rows == 1 && groups == 1)) {
        dequantize_kernel<T, FMT, true><<<grid, THREADS, 0, st>>>(codes, scales, rows, k, out);
    } else {
        constexpr int bytes = TILE * TILE * (int)sizeof(T);
        if (bytes > 48 * 1024 - TILE_BYTES) {
            const cudaError_t e = cudaFuncSetAttribute(dequantize_kernel<T, FMT, false>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
            if (e != cudaSuccess) return OZK_ERR_CUDA_BASE + (int)e;
        }
        dequantize_kernel<T, FMT, false><<<grid, THREADS, bytes, st>>>(codes, scales, rows, k, out);
    }
    OZK_CHECK_LAUNCH();
    return OZK_OK;
}

template <typename T>
int launch_dequantize(const uint8_t* codes, const uint8_t* scales, int fmt, int groups, int rows, int k, T* out,
                      cudaStream_t st) {
    return fmt == OZK_MX_E2M1 ? launch_dequantize_fmt<T, OZK_MX_E2M1>(codes, scales, groups, rows, k, out, st)
                              : launch_dequantize_fmt<T, OZK_MX_E4M3>(codes, scales, groups, rows, k, out, st);
}

}  // namespace

extern "C" size_t ozk_mx_code_bytes(int fmt, int groups, int rows, int k) {
    if (!fmt_ok(fmt) || groups < 1 || rows < 1 || rows > OZK_MX_ROWS_MAX || k < 1 || k > OZK_MX_KMAX) return 0;
    return (size_t)groups * rows * code_pitch(fmt, k);
}

extern "C" size_t ozk_mx_scale_bytes(int groups, int rows, int k) {
    if (groups < 1 || rows < 1 || rows > OZK_MX_ROWS_MAX || k < 1 || k > OZK_MX_KMAX) return 0;
    return (size_t)groups * scale_group_bytes(rows, k);
}

extern "C" int ozk_mx_quantize(const void* x, int dtype, int groups, int rows, int k, int64_t group_stride,
                               int64_t row_stride, int64_t k_stride, int fmt, int round_up, uint8_t* codes,
                               uint8_t* scales, ozk_stream_t stream) {
    if (!x || !codes || !scales || !fmt_ok(fmt) || groups < 1 || rows < 1 || rows > OZK_MX_ROWS_MAX || k < 1 ||
        k > OZK_MX_KMAX)
        return OZK_ERR_ARG;
    if (group_stride < 0 || row_stride < 0 || k_stride < 0 || !aligned16(codes) || !aligned16(scales)) return OZK_ERR_ARG;
    if (!dtype_ok(dtype) || !on_elements(x, dtype)) return OZK_ERR_ARG;
    if (tile_count(groups, rows, k) < 0) return OZK_ERR_ARG;
    QuantJob q = {};
    q.x = x;
    q.gs = groups == 1 ? 0 : group_stride;
    q.si = row_stride;
    q.sj = k == 1 ? 1 : k_stride;
    q.groups = groups;
    q.I = rows;
    q.J = k;
    q.row_codes = codes;
    q.row_scales = scales;
    return quantize(&q, 1, dtype, fmt, round_up != 0, reinterpret_cast<cudaStream_t>(stream));
}

namespace {

bool operand_ok(const uint8_t* p) { return p && (reinterpret_cast<uintptr_t>(p) & 31) == 0; }

// The job of x (rows x cols) with its operands, each one buffer of codes followed by scales, either of them absent
QuantJob job_of(const void* x, int rows, int cols, int64_t row_stride, int64_t col_stride, int fmt, uint8_t* along_rows,
                uint8_t* along_cols) {
    QuantJob q = {};
    q.x = x;
    q.si = row_stride;
    q.sj = cols == 1 ? 1 : col_stride;
    q.groups = 1;
    q.I = rows;
    q.J = cols;
    q.row_codes = along_rows;
    if (along_rows) q.row_scales = along_rows + rows * code_pitch(fmt, cols);
    q.col_codes = along_cols;
    if (along_cols) q.col_scales = along_cols + cols * code_pitch(fmt, rows);
    return q;
}

bool matrix_ok(const void* x, int dtype, int rows, int cols, int64_t rs, int64_t cs) {
    return x && dtype_ok(dtype) && on_elements(x, dtype) && rows >= 1 && cols >= 1 &&
           rows <= OZK_MX_KMAX && cols <= OZK_MX_KMAX && rs >= 0 && cs >= 0 && tile_count(1, rows, cols) > 0;
}

// C (m x n, contiguous) = A B^T for operands that are one buffer each
int product(const uint8_t* A, const uint8_t* B, int fmt, int m, int n, int k, void* C, int dtype, int32_t* err,
            ozk_stream_t stream) {
    const long long pitch = code_pitch(fmt, k);
    return ozk_mx_gemm(A, A + m * pitch, fmt, B, B + n * pitch, fmt, m, n, k, C, n, dtype, err, stream);
}

}  // namespace

extern "C" int ozk_mx_quantize_both(const void* x, int dtype, int rows, int cols, int64_t row_stride, int64_t col_stride,
                                    int fmt, int round_up, uint8_t* along_rows, uint8_t* along_cols,
                                    ozk_stream_t stream) {
    if (!matrix_ok(x, dtype, rows, cols, row_stride, col_stride) || !fmt_ok(fmt)) return OZK_ERR_ARG;
    if (!operand_ok(along_rows) || !operand_ok(along_cols)) return OZK_ERR_ARG;
    QuantJob q = job_of(x, rows, cols, row_stride, col_stride, fmt, along_rows, along_cols);
    return quantize(&q, 1, dtype, fmt, round_up != 0, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ozk_mx_linear_forward(const void* x, int x_dtype, int64_t x_row_stride, int64_t x_col_stride, const void* w,
                                     int w_dtype, int64_t w_row_stride, int64_t w_col_stride, int m, int n, int k, int fmt,
                                     int round_up, uint8_t* x_along_k, uint8_t* w_along_k, uint8_t* x_along_m,
                                     uint8_t* w_along_n, void* y, int32_t* err, ozk_stream_t stream) {
    if (!matrix_ok(x, x_dtype, m, k, x_row_stride, x_col_stride) || !matrix_ok(w, w_dtype, n, k, w_row_stride, w_col_stride))
        return OZK_ERR_ARG;
    if (!fmt_ok(fmt) || !operand_ok(x_along_k) || !operand_ok(w_along_k) || !y || !on_elements(y, x_dtype) || !err)
        return OZK_ERR_ARG;
    if ((x_along_m && !operand_ok(x_along_m)) || (w_along_n && !operand_ok(w_along_n))) return OZK_ERR_ARG;
    QuantJob q[2] = {job_of(x, m, k, x_row_stride, x_col_stride, fmt, x_along_k, x_along_m),
                           job_of(w, n, k, w_row_stride, w_col_stride, fmt, w_along_k, w_along_n)};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    int rc;
    if (x_dtype == w_dtype) {
        rc = quantize(q, 2, x_dtype, fmt, round_up != 0, st);
    } else {
        rc = quantize(q, 1, x_dtype, fmt, round_up != 0, st);
        if (rc == OZK_OK) rc = quantize(q + 1, 1, w_dtype, fmt, round_up != 0, st);
    }
    return rc != OZK_OK ? rc : product(x_along_k, w_along_k, fmt, m, n, k, y, x_dtype, err, stream);
}

extern "C" int ozk_mx_linear_backward(const void* dy, int dy_dtype, int64_t dy_row_stride, int64_t dy_col_stride,
                                      const uint8_t* x_along_m, const uint8_t* w_along_n, int m, int n, int k, int fmt,
                                      int round_up, uint8_t* dy_along_n, uint8_t* dy_along_m, void* dx, int dx_dtype,
                                      void* dw, int dw_dtype, int32_t* err, ozk_stream_t stream) {
    if (!matrix_ok(dy, dy_dtype, m, n, dy_row_stride, dy_col_stride) || !fmt_ok(fmt) || k < 1 || k > OZK_MX_KMAX || !err)
        return OZK_ERR_ARG;
    if (!dx && !dw) return OZK_ERR_ARG;
    if (!dtype_ok(dx_dtype) || !dtype_ok(dw_dtype) || !on_elements(dx, dx_dtype) || !on_elements(dw, dw_dtype)) return OZK_ERR_ARG;
    if (dx && (!operand_ok(w_along_n) || !operand_ok(dy_along_n))) return OZK_ERR_ARG;
    if (dw && (!operand_ok(x_along_m) || !operand_ok(dy_along_m))) return OZK_ERR_ARG;
    QuantJob q = job_of(dy, m, n, dy_row_stride, dy_col_stride, fmt, dx ? dy_along_n : nullptr, dw ? dy_along_m : nullptr);
    int rc = quantize(&q, 1, dy_dtype, fmt, round_up != 0, reinterpret_cast<cudaStream_t>(stream));
    if (rc == OZK_OK && dx) rc = product(dy_along_n, w_along_n, fmt, m, k, n, dx, dx_dtype, err, stream);
    if (rc == OZK_OK && dw) rc = product(dy_along_m, x_along_m, fmt, n, k, m, dw, dw_dtype, err, stream);
    return rc;
}

extern "C" int ozk_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int fmt, int groups, int rows, int k,
                                 void* out, int dtype, ozk_stream_t stream) {
    if (!codes || !scales || !out || !fmt_ok(fmt) || groups < 1 || rows < 1 || rows > OZK_MX_ROWS_MAX ||
        k < 1 || k > OZK_MX_KMAX)
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
