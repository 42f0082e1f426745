// Rows in 8 bits: writing rows into a store, reading them back, copying them between stores.
// Part of the single translation unit fps_kernels.cu (included there, in order).
//
// A row x of D elements is cut into blocks of 128.  With amax the largest finite magnitude of a block,
//   e    = the least integer with amax <= 448 * 2^e, at least -117        (448 = the largest e4m3 number)
//   code = e4m3(x * 2^-e), to nearest, ties to even; NaN and infinities become the NaN code
// so a scale is a power of two: x * 2^-e is exact, and so is code * 2^e in float32 and bfloat16 (4
// significant bits; e >= -117 keeps the smallest non-zero value, 2^-126, a normal float32).  The only
// rounding of a write is the one to e4m3 (relative 2^-4 in the normal range of the block).
#ifndef CORESETS_B200_ROWS8_STORE_CUH
#define CORESETS_B200_ROWS8_STORE_CUH

namespace {

constexpr int kR8Block = 128;       // elements that share a scale
constexpr int kR8MinExp = -117;

__host__ __device__ __forceinline__ int64_t r8_pitch(const int D) { return (D + 15) & ~15; }
__host__ __device__ __forceinline__ int r8_words(const int D) { return (D + 511) >> 9; }
// Byte offset of the scale word (4 consecutive blocks) w of a row: scales stand as the tensor core's
// scale-factor copy wants them, 512 bytes for 128 rows and 4 blocks, row 32 j + r at 16 r + 4 j.
__host__ __device__ __forceinline__ int64_t r8_scale_word(const int64_t row, const int w, const int words) {
    return ((row >> 7) * words + w) * 512 + ((row & 31) << 4) + (((row >> 5) & 3) << 2);
}

// 2^(b - 127) for a stored exponent byte; 255 stands for NaN
__device__ __forceinline__ float r8_scale_value(const unsigned b) {
    return __uint_as_float(b == 0u ? 0x00400000u : (b == 255u ? 0x7fc00000u : b << 23));
}
// products that keep subnormals (the translation unit is built with -ftz=true)
__device__ __forceinline__ float mul_keep(const float a, const float b) {
    float r;
    asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// two floats -> two codes (lo in the low byte)
__device__ __forceinline__ unsigned to_e4m3x2(const float lo, const float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 from_e4m3x2(const unsigned codes) {
    unsigned h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((unsigned short)codes));
    return __half22float2(*reinterpret_cast<const __half2*>(&h2));
}

__device__ __forceinline__ float r8_widen(const float v) { return v; }
__device__ __forceinline__ float r8_widen(const __half v) { return __half2float(v); }
__device__ __forceinline__ float r8_widen(const __nv_bfloat16 v) { return __uint_as_float((unsigned)__bfloat16_as_ushort(v) << 16); }

// 8 consecutive elements, 16-byte aligned
__device__ __forceinline__ void r8_load8(const float* p, float (&x)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void r8_load8(const T* p, float (&x)[8]) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
    const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned short lo = (unsigned short)(w[i] & 0xffffu), hi = (unsigned short)(w[i] >> 16);
        x[2 * i] = r8_widen(*reinterpret_cast<const T*>(&lo));
        x[2 * i + 1] = r8_widen(*reinterpret_cast<const T*>(&hi));
    }
}

// G lanes own a row (8 consecutive elements a lane and block); G < 16 serves rows of one block and 8 G
// elements at most.  U blocks are loaded before the first is worked on.  VEC: 16-byte loads (base and row stride 16-byte aligned, D a multiple of 8).
template <typename T, int G, int U, bool VEC>
__global__ void __launch_bounds__(kThreads) rows8_write_kernel(const cs_rows8 r, const T* __restrict__ X, const int64_t n,
                                                               const int64_t ld, const int64_t start) {
    const int D = r.dim, blocks = (D + kR8Block - 1) / kR8Block, words = r8_words(D);
    const int64_t pitch = r8_pitch(D);
    const int lane = threadIdx.x & 31, sub = lane & (G - 1);
    const int64_t per_pass = (int64_t)gridDim.x * (kThreads / G);
    // the whole warp takes the same number of passes: the shuffles below need all its lanes
    for (int64_t first = (int64_t)blockIdx.x * (kThreads / G) + (threadIdx.x >> 5) * (32 / G); first < n; first += per_pass) {
        const int64_t i = first + lane / G;
        const bool live = i < n;
        const T* src = X + (live ? i : 0) * ld;
        const int64_t row = start + (live ? i : 0);
        unsigned char* dst = reinterpret_cast<unsigned char*>(r.codes) + row * pitch;
        float norm = 0.0f;
        unsigned word = 0u;
        for (int b0 = 0; b0 < blocks; b0 += U) {
            float x[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = (b0 + u) * kR8Block + 8 * sub;
#pragma unroll
                for (int k = 0; k < 8; ++k) x[u][k] = 0.0f;
                if (VEC) {
                    if (live && c < D) r8_load8(src + c, x[u]);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (live && c + k < D) x[u][k] = r8_widen(src[c + k]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int b = b0 + u, c = b * kR8Block + 8 * sub;
                if (U > 1 && b >= blocks) break;
                unsigned top = 0u;         // magnitudes of finite numbers order like their bits
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const unsigned m = __float_as_uint(x[u][k]) & 0x7fffffffu;
                    if (m >= 0x7f800000u) x[u][k] = __uint_as_float(0x7fc00000u);
                    else top = m > top ? m : top;
                }
#pragma unroll
                for (int off = G / 2; off > 0; off >>= 1) {
                    const unsigned o = __shfl_xor_sync(kFull, top, off);
                    top = o > top ? o : top;
                }
                // amax = m * 2^E with 1 <= m < 2; 448 = 1.75 * 2^8
                int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
                e = e < kR8MinExp ? kR8MinExp : e;
                const float inv = __uint_as_float((unsigned)(127 - e) << 23), scale = __uint_as_float((unsigned)(127 + e) << 23);
                unsigned q[4];
                float sum = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    q[k] = to_e4m3x2(mul_keep(x[u][2 * k], inv), mul_keep(x[u][2 * k + 1], inv));
                    const float2 v = from_e4m3x2(q[k]);
                    sum = __fmaf_rn(v.x, v.x, sum);
                    sum = __fmaf_rn(v.y, v.y, sum);
                }
                norm = __fadd_rn(norm, __fmul_rn(__fmul_rn(sum, scale), scale));
                if (live && c < pitch) *reinterpret_cast<uint2*>(dst + c) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
                word |= (unsigned)(e + 127) << (8 * (b & 3));
                if ((b & 3) == 3 || b == blocks - 1) {
                    if (live && sub == 0)
                        *reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(r.scales) + r8_scale_word(row, b >> 2, words)) = word;
                    word = 0u;
                }
            }
        }
#pragma unroll
        for (int off = G / 2; off > 0; off >>= 1) norm = __fadd_rn(norm, __shfl_xor_sync(kFull, norm, off));
        if (live && sub == 0) r.norms[row] = norm;
    }
}

__device__ __forceinline__ void r8_narrow(float& o, const float v) { o = v; }
__device__ __forceinline__ void r8_narrow(__half& o, const float v) { o = __float2half_rn(v); }
__device__ __forceinline__ void r8_narrow(__nv_bfloat16& o, const float v) { o = __float2bfloat16_rn(v); }

// G lanes own an output row.  VEC: a lane turns 16 / sizeof(T) codes into one 16-byte store.
template <typename T, int G, bool VEC>
__global__ void __launch_bounds__(kThreads) rows8_read_kernel(const cs_rows8 r, const int64_t* __restrict__ rows, const int64_t m,
                                                              T* __restrict__ out, const int64_t ld) {
    constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;
    const int D = r.dim, words = r8_words(D);
    const int64_t pitch = r8_pitch(D);
    const int sub = threadIdx.x & (G - 1);
    const float nan = __uint_as_float(0x7fc00000u);
    for (int64_t i = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G; i < m; i += (int64_t)gridDim.x * (kThreads / G)) {
        const int64_t row = rows ? __ldg(rows + i) : i;
        const bool known = row >= 0 && row < r.count;
        const unsigned char* src = reinterpret_cast<const unsigned char*>(r.codes) + (known ? row : 0) * pitch;
        T* dst = out + i * ld;
        for (int c = sub * E; c < D; c += G * E) {
            float v[E];
            if (known) {
                const int b = c / kR8Block;
                const unsigned e = __ldg(reinterpret_cast<const unsigned char*>(r.scales) + r8_scale_word(row, b >> 2, words) + (b & 3));
                const float scale = r8_scale_value(e);
                if (E == 1) {
                    v[0] = mul_keep(from_e4m3x2(__ldg(src + c)).x, scale);
                } else {
                    unsigned w[2];
                    if (E == 8) {
                        const uint2 a = __ldg(reinterpret_cast<const uint2*>(src + c));
                        w[0] = a.x; w[1] = a.y;
                    } else {
                        w[0] = __ldg(reinterpret_cast<const unsigned*>(src + c)); w[1] = 0u;
                    }
#pragma unroll
                    for (int k = 0; k < E / 2; ++k) {
                        const float2 p = from_e4m3x2((w[k >> 1] >> (16 * (k & 1))) & 0xffffu);
                        v[(2 * k) % E] = mul_keep(p.x, scale);
                        v[(2 * k + 1) % E] = mul_keep(p.y, scale);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < E; ++k) v[k] = nan;
            }
            __align__(16) T o[E];
#pragma unroll
            for (int k = 0; k < E; ++k) r8_narrow(o[k], v[k]);
            if (VEC) __stcs(reinterpret_cast<uint4*>(dst + c), *reinterpret_cast<const uint4*>(o));
            else dst[c] = o[0];
        }
    }
}

// rows of one store appended to another as they are: codes, scales and norms; a row number outside
// the source becomes a row of NaN scales and a NaN norm.  One warp per row.
__global__ void __launch_bounds__(kThreads) rows8_take_kernel(const cs_rows8 src, const int64_t* __restrict__ rows, const int64_t m,
                                                              const cs_rows8 dst, const int64_t start) {
    const int D = src.dim, words = r8_words(D);
    const int64_t pitch = r8_pitch(D);
    const int lane = threadIdx.x & 31;
    for (int64_t i = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); i < m; i += (int64_t)gridDim.x * kWarps) {
        const int64_t row = __ldg(rows + i), to = start + i;
        const bool known = row >= 0 && row < src.count;
        const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(src.codes) + (known ? row : 0) * pitch);
        uint4* into = reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(dst.codes) + to * pitch);
        for (int c = lane; c < (int)(pitch >> 4); c += 32) into[c] = known ? __ldg(from + c) : make_uint4(0u, 0u, 0u, 0u);
        for (int w = lane; w < words; w += 32)
            *reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(dst.scales) + r8_scale_word(to, w, words)) =
                known ? __ldg(reinterpret_cast<const unsigned*>(reinterpret_cast<const unsigned char*>(src.scales) + r8_scale_word(row, w, words)))
                      : 0xffffffffu;
        if (lane == 0) dst.norms[to] = known ? __ldg(src.norms + row) : __uint_as_float(0x7fc00000u);
    }
}

}  // namespace

#endif  // CORESETS_B200_ROWS8_STORE_CUH
