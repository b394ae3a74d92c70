// ipx_mx4_kernels.h — rows in microscaled 4-bit floating point ("mx4"): quantisation, lookup, products, top-k search.
//
// The format (OCP microscaling, MXFP4). 32 consecutive elements of a row form a block with one power-of-two scale
// 2^s, s = max(floor(log2(largest magnitude)) - 2, -127), held as the byte s + 127; an element is an E2M1 code
// (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) of element / 2^s, rounded to nearest, ties to
// the even code, magnitudes beyond 6 to 6. A block with a NaN or an infinity has the scale byte 255 and stands for NaNs.
// A value code x 2^s has two significant bits and an exponent in fp32's (and bf16's) range: it is exact in both.
// 17 bytes per 32 elements: 408 bytes for 768 of them, where fp32 takes 3072 and bf16 1536.
//
// External form: codes [n][nb][16] bytes (element 2i of a block in the low nibble of byte i), scales [n][nb] bytes,
// nb = ceil(d / 32). Codes behind element d are 0.
//
// In the index the same bytes lie as the scaled MFMA wants them. v_mfma_scale_f32_32x32x64_f8f6f4 multiplies 32 rows by
// 32 columns over 64 elements: lane l holds row l & 31, elements 32 (l >> 5) .. + 31 — one whole block, 16 bytes, with
// one scale. So a K-set is 64 elements (two blocks) and
//   codes  [group of 32 rows][K-set][row][half][16 bytes]          one operand = one 1-KiB wave load
//   scales [group of 32 rows][row][quad of 4 K-sets][half][4 bytes]  one dword = the scales of a lane's next four operands
// Rows go from HBM straight into the registers of the one wave that multiplies them; LDS holds the queries only.
//
// Queries. The matrix core takes its two operands in different formats; fp32 queries are split into E2M3 parts (sign, two
// exponent bits, three mantissa bits, own scale per block and part): q = part_0 + part_1 + ... with each part the rounding of what
// the earlier ones left. E2M3 runs at the 4-bit rate (measured beside 4-bit rows: 5.9 PFLOP/s; E4M3, 4.2; two E2M1
// operands, 7.1). One part leaves 2^-5.1 of a Gaussian query (2-norm), two 2^-10.3, five 2^-26 (elementwise at most
// 2^-24 of the block's largest magnitude there, 2^-20 whatever the data).
#pragma once
#include "ipx_bf16_kernels.h"

namespace ipx {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int MX_GROUP = 32;             // rows per group
constexpr int MX_KSET = 64;              // elements per K-set
constexpr int MX_SET_BYTES = 1024;       // codes of one K-set of one group
constexpr int MX_THREADS = 512;          // 8 waves
constexpr int MX_RG = 2;                 // groups per wave tile
constexpr int MX_TILE = MX_RG * MX_GROUP;
constexpr int MX_SAMPLE = 8192;          // rows a search samples for its floor (mx4_floor_kernel)
constexpr int MX_DIRECT = 16384;         // indexes of up to this many rows are searched without a floor

__device__ __forceinline__ float mx_scale_f32(uint32_t byte) {          // 2^(byte - 127); 255: NaN
    return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}
// scale byte of a block from the largest magnitude's bits (sign cleared; NaN and inf order above all finite values)
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
__device__ __forceinline__ uint32_t mx_code(float x, float inv) {       // E2M1 code of x * inv
    const float a = fabsf(x) * inv;
    // steps of 0.5 below 2, of 1 below 4, of 2 beyond: the codes count the steps
    const float c = a < 2.f ? rintf(a * 2.f) : a < 4.f ? rintf(a) + 2.f : fminf(rintf(a * 0.5f) + 4.f, 7.f);
    return (uint32_t)(int)c | (__float_as_uint(x) >> 31 << 3);
}
// eight codes of one dword -> values before scaling, elements in order
__device__ __forceinline__ void mx_decode8(uint32_t w, float (&v)[8]) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = e[0]; v[7] = e[1];
}
// gid / np for gid < 2^32, 2 <= np < 2^32, magic = ceil(2^64 / np)
__device__ __forceinline__ uint32_t div_by(uint32_t gid, uint64_t magic) { return (uint32_t)__umul64hi((uint64_t)gid, magic); }

// where block b (32 elements) of row `row` lies in the index
__device__ __forceinline__ size_t mx_code_at(int64_t row, int b, int nks) {
    return ((size_t)(row >> 5) * nks + (b >> 1)) * MX_SET_BYTES + (row & 31) * 32 + (b & 1) * 16;
}
__device__ __forceinline__ size_t mx_scale_at(int64_t row, int b, int nkq) {
    return (((size_t)row * nkq + (b >> 3)) * 2 + (b & 1)) * 4 + ((b >> 1) & 3);
}

__device__ __forceinline__ void store_as(void* out, int dtype, size_t i, float v) {
    if (dtype == 0) ((float*)out)[i] = v;
    else if (dtype == 1) ((__half*)out)[i] = __float2half_rn(v);
    else ((uint16_t*)out)[i] = f32_to_bf16_rne(v);
}
// eight outputs; `wide`: they start at a multiple of 16 bytes
__device__ __forceinline__ void store8(void* out, int dtype, size_t i, const float (&v)[8], int count, bool wide) {
    if (wide && count == 8) {
        if (dtype == 0) {
            float4* o = (float4*)((float*)out + i);
            o[0] = make_float4(v[0], v[1], v[2], v[3]);
            o[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t lo, hi;
                if (dtype == 1) {
                    lo = __half_as_ushort(__float2half_rn(v[2 * e]));
                    hi = __half_as_ushort(__float2half_rn(v[2 * e + 1]));
                } else {
                    lo = f32_to_bf16_rne(v[2 * e]);
                    hi = f32_to_bf16_rne(v[2 * e + 1]);
                }
                w[e] = lo | hi << 16;
            }
            *(uint4*)((uint16_t*)out + i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < count) store_as(out, dtype, i + e, v[e]);
}

// ---- quantisation ----------------------------------------------------------------------------------------------
// Rows [n, d] (f32 / f16 / bf16, `stride` elements apart) -> codes and scales, in the external form or (INDEX) at rows
// row0.. of an index. Four adjacent lanes per block, eight elements each: the block's largest magnitude is two exchanges
// of lanes away, a wave reads 512 consecutive elements and writes 256 consecutive bytes. Bound by HBM.
template <bool INDEX>
__global__ void __launch_bounds__(256)
mx4_quantize_kernel(const void* __restrict__ src, int dtype, int64_t stride, uint32_t total, uint64_t magic, int np, int d,
                    bool wide, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t row0, int nks, int nkq) {
    const uint32_t gid = blockIdx.x * 256u + threadIdx.x;
    if (gid >= total) return;                               // a multiple of 4: the four lanes of a block stay together
    const uint32_t r = div_by(gid, magic);
    const int piece = (int)(gid - r * (uint32_t)np), e0 = piece * 8;
    const int64_t at = (int64_t)r * stride + e0;
    float x[8];
    if (wide && e0 + 8 <= d) {
        if (dtype == 0) {
            const float4 a = *(const float4*)((const float*)src + at), b = *(const float4*)((const float*)src + at + 4);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
            const uint4 w = *(const uint4*)((const uint16_t*)src + at);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint16_t u = (uint16_t)(ws[e >> 1] >> (16 * (e & 1)));
                x[e] = dtype == 1 ? __half2float(__ushort_as_half(u)) : __uint_as_float((uint32_t)u << 16);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = e0 + e < d ? load_as_f32(src, dtype, at + e) : 0.f;
    }
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));      // quad_perm [1,0,3,2]
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));      // quad_perm [2,3,0,1]
    const uint32_t byte = mx_scale_byte(top);
    const float inv = __uint_as_float((254u - byte) << 23);
    uint32_t w = 0;
    if (byte != 255)
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= mx_code(x[e], inv) << (4 * e);
    const int b = piece >> 2, p = piece & 3;
    if constexpr (INDEX) {
        const int64_t row = row0 + r;
        *(uint32_t*)(codes + mx_code_at(row, b, nks) + p * 4) = w;
        if (p == 0) scales[mx_scale_at(row, b, nkq)] = (uint8_t)byte;
    } else {
        const size_t blk = (size_t)r * (np >> 2) + b;
        *(uint32_t*)(codes + blk * 16 + p * 4) = w;
        if (p == 0) scales[blk] = (uint8_t)byte;
    }
}

// external form -> rows row0.. of an index; one thread per block
__global__ void __launch_bounds__(256)
mx4_place_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t total, uint64_t magic, int nb,
                 int d, uint8_t* __restrict__ X, uint8_t* __restrict__ Xs, int64_t row0, int nks, int nkq) {
    const uint32_t gid = blockIdx.x * 256u + threadIdx.x;
    if (gid >= total) return;
    const uint32_t r = nb == 1 ? gid : div_by(gid, magic);
    const int b = (int)(gid - r * (uint32_t)nb);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint8_t* s = codes + (size_t)gid * 16 + 4 * i;            // (the caller's bytes may start anywhere)
        w[i] = s[0] | (uint32_t)s[1] << 8 | (uint32_t)s[2] << 16 | (uint32_t)s[3] << 24;
        const int left = d - b * 32 - i * 8;                            // codes behind element d count as 0
        if (left < 8) w[i] &= left <= 0 ? 0u : (1u << (4 * left)) - 1u;
    }
    *(uint4*)(X + mx_code_at(row0 + r, b, nks)) = make_uint4(w[0], w[1], w[2], w[3]);
    Xs[mx_scale_at(row0 + r, b, nkq)] = scales[gid];
}

// external form -> values; one thread per eight elements
__global__ void __launch_bounds__(256)
mx4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t total, uint64_t magic,
                      int np, int d, int nb, void* __restrict__ out, int dtype, bool wide) {
    const uint32_t gid = blockIdx.x * 256u + threadIdx.x;
    if (gid >= total) return;
    const uint32_t r = np == 1 ? gid : div_by(gid, magic);
    const int piece = (int)(gid - r * (uint32_t)np);
    const size_t blk = (size_t)r * nb + (piece >> 2);
    const uint8_t* s = codes + blk * 16 + (piece & 3) * 4;
    const uint32_t w = wide ? *(const uint32_t*)s : s[0] | (uint32_t)s[1] << 8 | (uint32_t)s[2] << 16 | (uint32_t)s[3] << 24;
    const float sc = mx_scale_f32(scales[blk]);
    float v[8];
    mx_decode8(w, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= sc;
    const int left = d - piece * 8;
    store8(out, dtype, (size_t)r * d + piece * 8, v, left < 8 ? left : 8, wide);
}

// max |x|^2 over rows [row0, row0 + n) of an mx4 index, for the margin rule (rescore_kernel), as float bits. A row with a
// NaN block scores NaN in the scan and in the exact chain alike — it is never a candidate and never a result — so it does
// not enter the maximum; a sum that overflows does (as inf: every margin test then fails, which is intended).
// One wave per group of 32 rows: the loads of the scan.
__global__ void __launch_bounds__(256)
mx4_norm_max_kernel(const uint8_t* __restrict__ X, const uint8_t* __restrict__ Xs, int64_t row0, int64_t n, int nks, int nkq,
                    uint32_t* __restrict__ maxsq) {
    const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
    const int64_t g0 = row0 >> 5, g1 = (row0 + n + 31) >> 5;
    float best = 0.f;
    for (int64_t g = g0 + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); g < g1; g += (int64_t)gridDim.x * 4) {
        const int64_t row = g * 32 + l31;
        float acc = 0.f;
        for (int ks = 0; ks < nks; ++ks) {
            const uint4 c = *(const uint4*)(X + ((size_t)g * nks + ks) * MX_SET_BYTES + l31 * 32 + h * 16);
            const float sc = mx_scale_f32(Xs[mx_scale_at(row, 2 * ks + h, nkq)]);
            const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[8];
                mx_decode8(w[i], v);
#pragma unroll
                for (int e = 0; e < 8; ++e) { const float y = v[e] * sc; acc = fmaf(y, y, acc); }
            }
        }
        acc += __shfl_xor(acc, 32);
        if (row >= row0 && row < row0 + n && acc == acc) best = fmaxf(best, acc);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) best = fmaxf(best, __shfl_xor(best, off));
    if (lane == 0) atomicMax(maxsq, __float_as_uint(best));
}

// ---- lookup ----------------------------------------------------------------------------------------------------
// out[i] = scale[i] * row(ids[i]) for an index of any storage (xfmt 0: fp32 tiles of 128 rows, 1: bf16 tiles of 256, 2:
// mx4). One thread per eight elements of an output row. The product is rounded to fp32, then once to the output type.
// The empty slot id -1 gives a row of zeros; so does any other id outside the index, which also sets *err.
__global__ void __launch_bounds__(256)
lookup_kernel(const void* __restrict__ X, const uint8_t* __restrict__ Xs, int xfmt, int nks, int nkq, int64_t id_base, int64_t N,
              const int64_t* __restrict__ ids, const float* __restrict__ scale, uint32_t total, uint64_t magic, int np, int d,
              void* __restrict__ out, int dtype, bool wide, int* err) {
    const uint32_t gid = blockIdx.x * 256u + threadIdx.x;
    if (gid >= total) return;
    const uint32_t i = np == 1 ? gid : div_by(gid, magic);
    const int piece = (int)(gid - i * (uint32_t)np);
    const int64_t id = ids[i];
    const uint64_t row = (uint64_t)id - (uint64_t)id_base;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row < (uint64_t)N) {
        const float s = scale ? scale[i] : 1.f;
        if (xfmt == 2) {
            const int b = piece >> 2;
            const uint32_t w = *(const uint32_t*)((const uint8_t*)X + mx_code_at((int64_t)row, b, nks) + (piece & 3) * 4);
            const float sc = mx_scale_f32(Xs[mx_scale_at((int64_t)row, b, nkq)]);
            mx_decode8(w, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= sc;
        } else if (xfmt == 1) {
            const int64_t tile = (int64_t)row / HBD;
            const int rr = (int)(row - (uint64_t)tile * HBD), c = (piece & 3) ^ ((rr >> 2) & 3);
            const uint4 w = *(const uint4*)((const char*)X + (((size_t)tile * nks + (piece >> 2)) * HBD + rr) * 64 + c * 16);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[2 * e] = bf16_lo(ws[e]); v[2 * e + 1] = bf16_hi(ws[e]); }
        } else {
            const int64_t tile = (int64_t)row / BD;
            const int rr = (int)(row - (uint64_t)tile * BD), sw = (rr >> 2) & 3, c0 = (piece & 1) * 2;
            const char* line = (const char*)X + (((size_t)tile * nks + (piece >> 1)) * BD + rr) * 64;
            const f32x4 a = *(const f32x4*)(line + (c0 ^ sw) * 16), b = *(const f32x4*)(line + ((c0 + 1) ^ sw) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
        }
        if (scale)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= s;
    } else if (id != -1 && piece == 0) {
        *err = 1;
    }
    const int left = d - piece * 8;
    store8(out, dtype, (size_t)i * d + piece * 8, v, left < 8 ? left : 8, wide);
}

// ---- queries for the matrix core -------------------------------------------------------------------------------
// A packed query block of BQ queries, per quad of K-sets (256 elements) and part:
//   [K-set of the quad][half][query][16 bytes]   the first 16 bytes of the 32 codes, then
//   [K-set of the quad][half][query][8 bytes]    (E2M3 only) the last 8: 32 x 6 bits = 24 bytes, and
//   [half][query][4 bytes]                       the scales of the quad's four K-sets
// laid out so that a wave's LDS reads are contiguous and a quad is one contiguous copy.
constexpr int MX_E2M3 = 2, MX_E2M1 = 4;      // operand format numbers of the instruction
template <int FMT> __host__ __device__ constexpr int mx_code_bytes() { return FMT == MX_E2M3 ? 24 : 16; }
template <int FMT> __host__ __device__ constexpr int mx_part_bytes(int bq) { return bq * (8 * mx_code_bytes<FMT>() + 8); }

struct MxQueryInfo {      // of one query
    float sumsq;          // |q|^2                          (both 1e-37 larger where q has a nonzero element: squares of
    float restsq;         // |q - sum of its parts|^2        very small elements vanish, the bounds they stand for must not)
};

// One workgroup per query (rows beyond nq are written as zeros). Eight lanes per block, four elements each.
__global__ void __launch_bounds__(256)
mx4_pack_queries_kernel(const void* __restrict__ src, int dtype, int nq, int d, int parts, int bq, int nkq, uint8_t* __restrict__ dst,
                        MxQueryInfo* __restrict__ info, int* __restrict__ todo) {
    __shared__ float red[8];
    const int tid = threadIdx.x, lane = tid & 63;
    bool nonzero = false;
    const int64_t q = blockIdx.x;
    const int part_bytes = bq * 200;
    uint8_t* block = dst + (size_t)(q / bq) * nkq * parts * part_bytes;
    const int ql = (int)(q % bq), sub = tid & 7;
    float ss = 0.f, rr = 0.f;
    for (int b = tid >> 3; b < nkq * 8; b += 32) {                      // block b: K-set b >> 1, half b & 1
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = b * 32 + sub * 4 + e;
            x[e] = q < nq && at < d ? load_as_f32(src, dtype, q * (int64_t)d + at) : 0.f;
            ss = fmaf(x[e], x[e], ss);
            nonzero |= x[e] != 0.f;
        }
        const int quad = b >> 3, j = (b >> 1) & 3, h = b & 1;
        for (int p = 0; p < parts; ++p) {
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
            const bool bad = top >= 0x7f800000u;                        // NaN / inf: the block's scale is NaN
            // smallest s with the largest magnitude <= 7.5 x 2^s
            int s = -127;
            if (!bad && top) {
                int ex;
                const float m = frexpf(__uint_as_float(top), &ex);      // m 2^ex, 0.5 <= m < 1
                s = max(ex - 3 + (m > 0.9375f ? 1 : 0), -127);
            }
            uint32_t bits = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (bad) { x[e] = 0.f; continue; }
                const float a = ldexpf(fabsf(x[e]), -s);
                // codes count steps of 1/8 below 2, 1/4 below 4, 1/2 up to 7.5
                const int c = a < 2.f ? (int)rintf(a * 8.f) : a < 4.f ? (int)rintf(a * 4.f) + 8 : min((int)rintf(a * 2.f) + 16, 31);
                const float v = c < 16 ? c * 0.125f : c < 24 ? (c - 8) * 0.25f : (c - 16) * 0.5f;
                const uint32_t neg = __float_as_uint(x[e]) >> 31;
                bits |= ((uint32_t)c | neg << 5) << (6 * e);
                x[e] -= ldexpf(neg ? -v : v, s);                        // exact: both are multiples of x's last place
            }
            uint8_t* part = block + ((size_t)quad * parts + p) * part_bytes;
            // the lane's 24 bits are bytes 3 sub .. 3 sub + 2 of the block's 24
#pragma unroll
            for (int y = 0; y < 3; ++y) {
                const int at = sub * 3 + y;
                uint8_t* o = at < 16 ? part + ((j * 2 + h) * bq + ql) * 16 + at
                                     : part + bq * 128 + ((j * 2 + h) * bq + ql) * 8 + (at - 16);
                *o = (uint8_t)(bits >> (8 * y));
            }
            if (sub == 0) part[bq * 192 + (h * bq + ql) * 4 + j] = bad ? 255 : (uint8_t)(s + 127);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) rr = fmaf(x[e], x[e], rr);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { ss += __shfl_xor(ss, off); rr += __shfl_xor(rr, off); }
    if (lane == 0) { red[tid >> 6] = ss; red[4 + (tid >> 6)] = rr; }
    const float least = __syncthreads_or(nonzero) ? 1e-37f : 0.f;
    if (tid == 0 && q < nq) {
        info[q] = {red[0] + red[1] + red[2] + red[3] + least, red[4] + red[5] + red[6] + red[7] + least};
        if (todo) todo[q] = 0;
    }
}

// external mx4 rows as queries (one part, E2M1); one thread per block of every padded query
__global__ void __launch_bounds__(256)
mx4_pack_codes_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int nq, int d, int bq, int nkq,
                      int64_t total, uint8_t* __restrict__ dst) {
    const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (gid >= total) return;
    const int64_t q = gid / (nkq * 8);
    const int b = (int)(gid - q * (nkq * 8)), nb = (d + 31) / 32;
    uint32_t w[4] = {0, 0, 0, 0};
    uint8_t sc = 0;
    if (q < nq && b < nb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint8_t* s = codes + ((size_t)q * nb + b) * 16 + 4 * i;
            w[i] = s[0] | (uint32_t)s[1] << 8 | (uint32_t)s[2] << 16 | (uint32_t)s[3] << 24;
            const int left = d - b * 32 - i * 8;
            if (left < 8) w[i] &= left <= 0 ? 0u : (1u << (4 * left)) - 1u;
        }
        sc = scales[(size_t)q * nb + b];
    }
    const int part_bytes = bq * 136, quad = b >> 3, j = (b >> 1) & 3, h = b & 1, ql = (int)(q % bq);
    uint8_t* part = dst + ((size_t)(q / bq) * nkq + quad) * part_bytes;
    *(uint4*)(part + ((j * 2 + h) * bq + ql) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    part[bq * 128 + (h * bq + ql) * 4 + j] = sc;
}

// ---- products --------------------------------------------------------------------------------------------------
struct MxParams {
    const uint8_t* X;            // index codes
    const uint8_t* Xs;           // index scales
    const uint8_t* Q;            // packed query blocks
    int64_t N;                   // rows of the index
    int nq, d, nks, nkq;
    int S;                       // splits: workgroups that share a query block
    int qc;                      // quads of the query block that LDS holds at a time (nkq: all, staged once)
    int64_t g0, gstep;           // wave tile t covers groups g0 + t * gstep, + 1
    int64_t ntiles;
    // scores
    float* out;                  // [nq][ld]
    int64_t ld, row0, n;         // columns 0 .. n - 1 are rows row0 ..; row0 < 0: column = 64 t + row of the tile
    const void* q;               // the caller's queries (recomputation of those with NaN / inf elements), or null
    int q_dtype;
    const MxQueryInfo* info;
    // search
    const float* tau;            // [nq] floor: a hit scores above it, or equals it with row < row_below
    const int64_t* row_below;    // [nq]
    uint64_t* cand;              // [nq][S][cap] keys of the hits
    int* cnt;                    // [nq][S]
    int* todo;                   // [nq] set to 1 when a list overflows
    int cap;
};

// <q, row> as a chain of fp32 fmafs: queries with NaN or infinite elements (the parts hold neither)
__device__ __forceinline__ float mx4_plain_dot(const MxParams& p, int q, int64_t row) {
    float acc = 0.f;
#pragma unroll 1
    for (int e = 0; e < p.d; ++e) {
        const int b = e >> 5;
        const uint32_t code = (p.X[mx_code_at(row, b, p.nks) + ((e & 31) >> 1)] >> (4 * (e & 1))) & 15;
        const uint32_t m = code & 7;
        const float v = (m < 4 ? m * 0.5f : m < 6 ? m - 2.f : 2.f * m - 8.f) * mx_scale_f32(p.Xs[mx_scale_at(row, b, p.nkq)]);
        acc = fmaf(code & 8 ? -v : v, load_as_f32(p.q, p.q_dtype, (int64_t)q * p.d + e), acc);
    }
    return acc;
}

enum { MX_SCORES = 0, MX_SEARCH = 1 };

// One wave: 64 rows (two groups) x BQ = 32 CG queries; 8 waves a workgroup, which share the query block in LDS and nothing
// else: while the whole block fits (qc == nkq) the main loop has no barrier. A quad of K-sets (256 elements) is the step of
// the loop: its row operands were fetched one step earlier (across tiles too), and per K-set, part and pair of 32 x 32
// blocks one MFMA runs. Tiles are dealt round-robin over the waves of a query block's S workgroups.
// When the query block does not fit, its quads go through LDS qc at a time, all waves in step.
template <int CG, int PARTS, int FMT, int MODE>
__global__ void __launch_bounds__(MX_THREADS)
mx4_product_kernel(const MxParams p) {
    constexpr int BQ = 32 * CG, PART = mx_part_bytes<FMT>(BQ), QUAD = PARTS * PART;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int* cnts = (int*)(smem + (size_t)p.qc * QUAD);                    // [BQ]  (MX_SEARCH)
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nqb = (int)gridDim.x / p.S;
    // consecutive logical ids sit on one XCD: the query blocks of one split side by side, so that its L2 serves their
    // common rows once
    const int logical = xcd_remap(blockIdx.x, gridDim.x);
    const int split = logical / nqb, qb = logical - split * nqb;
    const char* qblock = (const char*)p.Q + (size_t)qb * p.nkq * QUAD;

    float tau[CG];
    int64_t below[CG];
    if constexpr (MODE == MX_SEARCH) {
#pragma unroll
        for (int c = 0; c < CG; ++c) {
            const int q = qb * BQ + c * 32 + l31;
            tau[c] = q < p.nq ? p.tau[q] : INFINITY;
            below[c] = q < p.nq ? p.row_below[q] : 0;
        }
        for (int i = tid; i < BQ; i += MX_THREADS) cnts[i] = 0;
    }
    int redo = 0;                                                       // MX_SCORES: this lane's queries that are not finite
    if constexpr (MODE == MX_SCORES) {
        if (p.q)
#pragma unroll
            for (int c = 0; c < CG; ++c) {
                const int q = qb * BQ + c * 32 + l31;
                if (q < p.nq && !(p.info[q].sumsq <= FLT_MAX)) redo |= 1 << c;
            }
    }
    auto stage = [&](int quad0) {
        const int n16 = (p.nkq - quad0 < p.qc ? p.nkq - quad0 : p.qc) * (QUAD / 16);
        const uint4* s = (const uint4*)(qblock + (size_t)quad0 * QUAD);
        for (int i = tid; i < n16; i += MX_THREADS) ((uint4*)smem)[i] = s[i];
    };
    const bool resident = p.qc >= p.nkq;
    if (resident) stage(0);
    __syncthreads();

    const int64_t per_round = (int64_t)p.S * 8;
    const int64_t rounds = (p.ntiles + per_round - 1) / per_round;
    const int64_t tile0 = (int64_t)split * 8 + wave;
    const size_t group_bytes = (size_t)p.nks * MX_SET_BYTES, group_scales = (size_t)p.nkq * 256;

    struct Operands { uint4 a[4][MX_RG]; uint32_t s[MX_RG]; };
    Operands A0, A1;
    auto fetch = [&](Operands& o, int64_t tile, int quad) {
        if (tile >= p.ntiles) return;
        const int64_t g = p.g0 + tile * p.gstep;
#pragma unroll
        for (int r = 0; r < MX_RG; ++r) {
            const uint8_t* x = p.X + (size_t)(g + r) * group_bytes + (size_t)quad * 4 * MX_SET_BYTES + l31 * 32 + h * 16;
            o.s[r] = *(const uint32_t*)(p.Xs + (size_t)(g + r) * group_scales + (size_t)l31 * p.nkq * 8 + quad * 8 + h * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (quad * 4 + j < p.nks) o.a[j][r] = *(const uint4*)(x + j * MX_SET_BYTES);
        }
    };

    f32x16 acc[MX_RG][CG];
    auto clear = [&]() {
#pragma unroll
        for (int r = 0; r < MX_RG; ++r)
#pragma unroll
            for (int c = 0; c < CG; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[r][c][i] = 0.f;
    };
    clear();

    auto multiply = [&](const Operands& o, int quad) {
        const char* qq = smem + (size_t)(quad % p.qc) * QUAD;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            uint32_t qs[CG];
#pragma unroll
            for (int c = 0; c < CG; ++c)
                qs[c] = *(const uint32_t*)(qq + part * PART + BQ * 8 * mx_code_bytes<FMT>() + (h * BQ + c * 32 + l31) * 4);
            auto kset = [&](auto jc) {
                constexpr int j = decltype(jc)::value;
                if (quad * 4 + j >= p.nks) return;
#pragma unroll
                for (int c = 0; c < CG; ++c) {
                    const char* at = qq + part * PART + ((j * 2 + h) * BQ + c * 32 + l31) * 16;
                    const uint4 lo = *(const uint4*)at;
                    i32x8 b = {(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, 0, 0, 0, 0};
                    if constexpr (FMT == MX_E2M3) {
                        const uint2 hi = *(const uint2*)(qq + part * PART + BQ * 128 + ((j * 2 + h) * BQ + c * 32 + l31) * 8);
                        b[4] = (int)hi.x;
                        b[5] = (int)hi.y;
                    }
#pragma unroll
                    for (int r = 0; r < MX_RG; ++r) {
                        const i32x8 a = {(int)o.a[j][r].x, (int)o.a[j][r].y, (int)o.a[j][r].z, (int)o.a[j][r].w, 0, 0, 0, 0};
                        acc[r][c] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, acc[r][c], MX_E2M1, FMT, j, (int)o.s[r], j, (int)qs[c]);
                    }
                }
            };
            kset(std::integral_constant<int, 0>{});
            kset(std::integral_constant<int, 1>{});
            kset(std::integral_constant<int, 2>{});
            kset(std::integral_constant<int, 3>{});
        }
    };

    // column of the lane's first row in group r of a tile (MX_SCORES)
    auto column = [&](int64_t tile, int r) {
        return (p.row0 < 0 ? tile * MX_TILE + r * 32 : (p.g0 + tile * p.gstep + r) * 32 - p.row0) + 4 * h;
    };
    auto finish = [&](int64_t tile) {
        const int64_t g = p.g0 + tile * p.gstep;
#pragma unroll
        for (int c = 0; c < CG; ++c) {
            const int ql = c * 32 + l31, q = qb * BQ + ql;
            if constexpr (MODE == MX_SCORES) {
                if (q >= p.nq) continue;
#pragma unroll
                for (int r = 0; r < MX_RG; ++r) {
                    const int64_t col0 = column(tile, r);
                    float* o = p.out + (size_t)q * p.ld;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int64_t col = col0 + 8 * i;
                        const f32x4 v = {acc[r][c][4 * i], acc[r][c][4 * i + 1], acc[r][c][4 * i + 2], acc[r][c][4 * i + 3]};
                        if (col >= 0 && col + 4 <= p.n) {
                            __builtin_memcpy(o + col, &v, 16);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (col + e >= 0 && col + e < p.n) o[col + e] = v[e];
                        }
                    }
                }
            } else {
#pragma unroll
                for (int r = 0; r < MX_RG; ++r) {
                    float g4[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        g4[i] = fmaxf(fmaxf(acc[r][c][4 * i], acc[r][c][4 * i + 1]), fmaxf(acc[r][c][4 * i + 2], acc[r][c][4 * i + 3]));
                    if (!__any(fmaxf(fmaxf(g4[0], g4[1]), fmaxf(g4[2], g4[3])) >= tau[c])) continue;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (!__any(g4[i] >= tau[c])) continue;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float sc = acc[r][c][4 * i + e];
                            const int64_t doc = (g + r) * 32 + 4 * h + 8 * i + e;
                            if ((sc > tau[c] || (sc == tau[c] && doc < below[c])) && doc < p.N) {
                                const int pos = atomicAdd(&cnts[ql], 1);
                                if (pos < p.cap) p.cand[((size_t)q * p.S + split) * p.cap + pos] = make_key(sc, (uint32_t)doc);
                            }
                        }
                    }
                }
            }
        }
        if constexpr (MODE == MX_SCORES)
            if (__any(redo != 0)) {
#pragma unroll 1
                for (int i = 0; i < CG * MX_RG * 16; ++i) {
                    const int c = i / (MX_RG * 16), r = (i >> 4) % MX_RG, at = (i & 3) + 8 * ((i >> 2) & 3);
                    const int64_t col = column(tile, r) + at;
                    const int q = qb * BQ + c * 32 + l31;
                    if ((redo >> c & 1) && col >= 0 && col < p.n) p.out[(size_t)q * p.ld + col] = mx4_plain_dot(p, q, (g + r) * 32 + 4 * h + at);
                }
            }
    };

    // the flattened sequence of (round, quad) steps
    int64_t round = 0;
    int quad = 0;
    fetch(A0, tile0, 0);
    auto step = [&](Operands& cur, Operands& nxt) -> bool {            // false: that was the last one
        const int64_t tile = tile0 + round * per_round;
        if (!resident && quad % p.qc == 0) {
            __syncthreads();
            stage(quad);
            __syncthreads();
        }
        const bool last = quad + 1 == p.nkq;
        const int64_t nround = last ? round + 1 : round;
        const int nquad = last ? 0 : quad + 1;
        if (nround < rounds) fetch(nxt, tile0 + nround * per_round, nquad);
        if (tile < p.ntiles) {
            multiply(cur, quad);
            if (last) {
                finish(tile);
                clear();
            }
        }
        round = nround;
        quad = nquad;
        return round < rounds;
    };
    if (rounds > 0)
        while (step(A0, A1) && step(A1, A0)) {}

    if constexpr (MODE == MX_SEARCH) {
        __syncthreads();
        for (int i = tid; i < BQ; i += MX_THREADS) {
            const int q = qb * BQ + i;
            if (q >= p.nq) continue;
            const int n = cnts[i];
            p.cnt[(size_t)q * p.S + split] = n < p.cap ? n : p.cap;
            if (n > p.cap) p.todo[q] = 1;
        }
    }
}

// ---- the floor of a search -------------------------------------------------------------------------------------
// A search scores a sample of the index first (MX_SAMPLE rows, whole tiles at equal distances) and takes its j-th best
// score as the floor every hit has to reach: with j well above the share of the wanted list that falls into the sample,
// about j / sample of the index passes (the host chooses j: mx4_floor_rank), which is a few times the list. Equal scores
// are ordered by row as everywhere: where the j-th best sits among equals, rows up to its share of the index pass.
// One workgroup of 1024 per query: radix selection, 8 bits a pass, on the scores held in registers.
__global__ void __launch_bounds__(1024)
mx4_floor_kernel(const float* __restrict__ sample, int m, int j, int64_t N, float* __restrict__ tau, int64_t* __restrict__ row_below) {
    constexpr int PER = MX_SAMPLE / 1024;
    __shared__ int hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need, s_wave[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t q = blockIdx.x;
    uint32_t v[PER];                                           // entries tid * PER .. + PER - 1: a thread's are neighbours
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = tid * PER + i;
        const float s = e < m ? sample[q * (int64_t)m + e] : -INFINITY;
        v[i] = s > -FLT_MAX ? f32_ordered(s) : 0u;             // NaN and -inf are never hits
    }
    if (tid == 0) { s_prefix = 0; s_need = j; }
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (v[i] && (shift == 24 || (v[i] >> (shift + 8)) == (prefix >> (shift + 8)))) atomicAdd(&hist[(v[i] >> shift) & 255], 1);
        __syncthreads();
        if (wave == 0) {
            // the bucket that holds the need-th largest: lane l owns buckets 255 - 4 l .. 252 - 4 l
            int mine[4], sum = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) { mine[u] = hist[255 - 4 * lane - u]; sum += mine[u]; }
            int run = sum;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) { const int x = __shfl_up(run, off); if (lane >= off) run += x; }
            const int need = s_need;
            int before = run - sum;
            const bool here = before < need && run >= need;
            if (here) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (before < need && before + mine[u] >= need) {
                        s_prefix = prefix | (uint32_t)(255 - 4 * lane - u) << shift;
                        s_need = need - before;
                        before = 0x7fffffff;                   // found
                    } else if (before != 0x7fffffff) {
                        before += mine[u];
                    }
                }
            }
            if (!__any(here) && lane == 0) { s_prefix = 0; s_need = 0; }      // fewer than j numbers in the sample
        }
        __syncthreads();
        if (s_need == 0) break;
    }
    const uint32_t t = s_prefix;
    const int need = s_need;                                   // the need-th of the entries equal to t, in row order
    if (need == 0) {
        if (tid == 0) { tau[q] = -FLT_MAX; row_below[q] = 0; }
        return;
    }
    int eq = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) eq += v[i] == t ? 1 : 0;
    int run = eq;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) { const int x = __shfl_up(run, off); if (lane >= off) run += x; }
    if (lane == 63) s_wave[wave] = run;
    __syncthreads();
    int before = run - eq;
    for (int w = 0; w < wave; ++w) before += s_wave[w];
    if (before < need && before + eq >= need) {
        int k = before;
        for (int i = 0; i < PER; ++i)
            if (v[i] == t && ++k == need) {
                tau[q] = f32_unordered(t);
                row_below[q] = ((int64_t)(tid * PER + i + 1) * N + m - 1) / m;
            }
    }
}

// an index that is searched without a sample: every row that is a number is a hit
__global__ void __launch_bounds__(256)
mx4_no_floor_kernel(int nq, float* __restrict__ tau, int64_t* __restrict__ row_below) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < nq) { tau[i] = -FLT_MAX; row_below[i] = 0; }
}

}  // namespace ipx
