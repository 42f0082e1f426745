// Rows in 8 bits: writing rows into a store, reading them back, copying them between stores.
// Part of the single translation unit fps_kernels.cu (included there, in order).
//
// A row x of D elements is cut into blocks of 128.  With amax the largest finite magnitude of a block,
//   e    = the least integer with amax <= 448 * 2^e, at least -117        (448 = the largest e4m3 number)
//   code = e4m3(x * 2^-e), to nearest, ties to even; NaN and infinities become the NaN code
// so a scale is a power of two: x * 2^-e is exact, and so is code * 2^e in float32 and bfloat16 (4
// significant bits; e >= -117 keeps the smallest non-zero value, 2^-126, a normal float32).  The only
// rounding of a write is the one to e4m3 (relative 2^-4 in the normal range of the block).  Magnitudes of 248 * 2^120 and
// more round to 256 * 2^120, past float32: such a code reads as infinity.
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
__device__ __forceinline__ __half2 half_from_e4m3x2(const unsigned codes) {
    unsigned h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((unsigned short)codes));
    return *reinterpret_cast<const __half2*>(&h2);
}
__device__ __forceinline__ float2 from_e4m3x2(const unsigned codes) { return __half22float2(half_from_e4m3x2(codes)); }

__device__ __forceinline__ float r8_widen(const float v) { return v; }
__device__ __forceinline__ float r8_widen(const __half v) { return __half2float(v); }
__device__ __forceinline__ float r8_widen(const __nv_bfloat16 v) { return __uint_as_float((unsigned)__bfloat16_as_ushort(v) << 16); }

// V bytes of memory as whole elements, widened (narrow loads share lines with the next ones: those are kept)
template <typename T, int V>
__device__ __forceinline__ void r8_load(const T* p, float* x) {
    if constexpr (V == 16) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
        const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                x[i] = __uint_as_float(w[i]);
            } else {
                const unsigned short lo = (unsigned short)(w[i] & 0xffffu), hi = (unsigned short)(w[i] >> 16);
                x[2 * i] = r8_widen(*reinterpret_cast<const T*>(&lo));
                x[2 * i + 1] = r8_widen(*reinterpret_cast<const T*>(&hi));
            }
        }
    } else if constexpr (V == 8 && sizeof(T) == 4) {
        const float2 a = __ldg(reinterpret_cast<const float2*>(p));
        x[0] = a.x;
        x[1] = a.y;
    } else if constexpr (V == 4 && sizeof(T) == 2) {
        const unsigned w = __ldg(reinterpret_cast<const unsigned*>(p));
        const unsigned short lo = (unsigned short)(w & 0xffffu), hi = (unsigned short)(w >> 16);
        x[0] = r8_widen(*reinterpret_cast<const T*>(&lo));
        x[1] = r8_widen(*reinterpret_cast<const T*>(&hi));
    } else {
        static_assert(V == sizeof(T), "one element");
        x[0] = r8_widen(__ldg(p));
    }
}
// 8 consecutive elements from element c of a row of D, zeros behind its end (D is whole loads)
template <typename T, int V>
__device__ __forceinline__ void r8_load8(const T* row, const int c, const int D, const bool live, float (&x)[8]) {
    constexpr int E = V / (int)sizeof(T);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k += E)
        if (live && c + k < D) r8_load<T, V>(row + c + k, x + k);
}

// One block of a row in the registers of G lanes, 8 elements each: the codes of this lane, the exponent byte, this lane's part of the
// squared norm.
template <int G>
__device__ __forceinline__ uint2 r8_quantise(float (&x)[8], unsigned& byte, float& part) {
    unsigned top = 0u;                     // magnitudes order like their bits
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const unsigned m = __float_as_uint(x[k]) & 0x7fffffffu;
        top = m > top ? m : top;
    }
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) {
        const unsigned o = __shfl_xor_sync(kFull, top, off);
        top = o > top ? o : top;
    }
    if (__any_sync(kFull, top >= 0x7f800000u)) {
        // a NaN or an infinity somewhere in the warp's blocks: they become NaN and count for no maximum
        top = 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const unsigned m = __float_as_uint(x[k]) & 0x7fffffffu;
            if (m >= 0x7f800000u) x[k] = __uint_as_float(0x7fc00000u);
            else top = m > top ? m : top;
        }
#pragma unroll
        for (int off = G / 2; off > 0; off >>= 1) {
            const unsigned o = __shfl_xor_sync(kFull, top, off);
            top = o > top ? o : top;
        }
    }
    // amax = m * 2^E with 1 <= m < 2; 448 = 1.75 * 2^8
    int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = e < kR8MinExp ? kR8MinExp : e;
    const float inv = __uint_as_float((unsigned)(127 - e) << 23), scale = __uint_as_float((unsigned)(127 + e) << 23);
    unsigned q[4];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        q[k] = to_e4m3x2(mul_keep(x[2 * k], inv), mul_keep(x[2 * k + 1], inv));
        const __half2 v = half_from_e4m3x2(q[k]);          // (a half holds every code: the squares are exact)
        sum = fma_half(__low2half(v), __low2half(v), sum);
        sum = fma_half(__high2half(v), __high2half(v), sum);
    }
    byte = (unsigned)(e + 127);
    part = __fmul_rn(__fmul_rn(sum, scale), scale);
    return make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
}

// Bound by HBM.  G lanes own a row, 8 consecutive elements a lane and block; G < 16 serves rows of 8 G elements at
// most.  What a lane has in flight decides the rate, so U blocks are loaded before the first is worked on: of one row, or
// (ROWS, rows of one block) of U rows.  V: bytes of a load.
template <typename T, int G, int U, bool ROWS, int V>
__global__ void __launch_bounds__(kThreads) rows8_write_kernel(const cs_rows8 r, const T* __restrict__ X, const int64_t n,
                                                               const int64_t ld, const int64_t start) {
    const int D = r.dim, blocks = (D + kR8Block - 1) / kR8Block, words = r8_words(D);
    const int64_t pitch = r8_pitch(D);
    const int lane = threadIdx.x & 31, sub = lane & (G - 1);
    const int64_t per_pass = (int64_t)gridDim.x * (kThreads / G);
    unsigned char* codes = reinterpret_cast<unsigned char*>(r.codes);
    unsigned char* scales = reinterpret_cast<unsigned char*>(r.scales);
    // the whole warp takes the same number of passes: the shuffles need all its lanes
    for (int64_t first = (int64_t)blockIdx.x * (kThreads / G) + (threadIdx.x >> 5) * (32 / G); first < n; first += per_pass * (ROWS ? U : 1)) {
        float x[U][8], norm = 0.0f;
        if (ROWS) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t i = first + u * per_pass + lane / G;
                r8_load8<T, V>(X + (i < n ? i : 0) * ld, 8 * sub, D, i < n, x[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t i = first + u * per_pass + lane / G, row = start + i;
                unsigned byte;
                const uint2 q = r8_quantise<G>(x[u], byte, norm);
#pragma unroll
                for (int off = G / 2; off > 0; off >>= 1) norm = __fadd_rn(norm, __shfl_xor_sync(kFull, norm, off));
                if (i < n) {
                    if (8 * sub < pitch) *reinterpret_cast<uint2*>(codes + row * pitch + 8 * sub) = q;
                    if (sub == 0) {
                        *reinterpret_cast<unsigned*>(scales + r8_scale_word(row, 0, 1)) = byte;
                        r.norms[row] = norm;
                    }
                }
            }
        } else {
            const int64_t i = first + lane / G, row = start + i;
            const bool live = i < n;
            const T* src = X + (live ? i : 0) * ld;
            unsigned word = 0u;
            for (int b0 = 0; b0 < blocks; b0 += U) {
#pragma unroll
                for (int u = 0; u < U; ++u) r8_load8<T, V>(src, (b0 + u) * kR8Block + 8 * sub, D, live, x[u]);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int b = b0 + u, c = b * kR8Block + 8 * sub;
                    if (b >= blocks) break;
                    unsigned byte;
                    float part;
                    const uint2 q = r8_quantise<G>(x[u], byte, part);
                    norm = __fadd_rn(norm, part);
                    if (live && c < pitch) *reinterpret_cast<uint2*>(codes + row * pitch + c) = q;
                    word |= byte << (8 * (b & 3));
                    if ((b & 3) == 3 || b == blocks - 1) {
                        if (live && sub == 0) *reinterpret_cast<unsigned*>(scales + r8_scale_word(row, b >> 2, words)) = word;
                        word = 0u;
                    }
                }
            }
#pragma unroll
            for (int off = G / 2; off > 0; off >>= 1) norm = __fadd_rn(norm, __shfl_xor_sync(kFull, norm, off));
            if (live && sub == 0) r.norms[row] = norm;
        }
    }
}

__device__ __forceinline__ void r8_narrow(float& o, const float v) { o = v; }
__device__ __forceinline__ void r8_narrow(__half& o, const float v) { o = __float2half_rn(v); }
__device__ __forceinline__ void r8_narrow(__nv_bfloat16& o, const float v) { o = __float2bfloat16_rn(v); }

// Bound by HBM.  G lanes own a row; E codes a lane make one store of up to 16 bytes; R rows are in flight.
template <typename T, int E, int G, int R>
__global__ void __launch_bounds__(kThreads) rows8_read_kernel(const cs_rows8 r, const int64_t* __restrict__ rows, const int64_t m,
                                                              T* __restrict__ out, const int64_t ld) {
    const int D = r.dim, words = r8_words(D), sub = threadIdx.x & (G - 1);
    const int64_t pitch = r8_pitch(D), groups = (int64_t)gridDim.x * (kThreads / G);
    for (int64_t first = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G; first < m; first += groups * R) {
        const unsigned char* src[R];
        const unsigned char* sf[R];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int64_t i = first + u * groups, row = i < m ? (rows ? __ldg(rows + i) : i) : -1;
            const bool known = row >= 0 && row < r.count;
            src[u] = known ? reinterpret_cast<const unsigned char*>(r.codes) + row * pitch : nullptr;
            sf[u] = reinterpret_cast<const unsigned char*>(r.scales) + (known ? r8_scale_word(row, 0, words) : 0);
        }
        for (int c = sub * E; c < D; c += G * E) {
            uint2 code[R];
            unsigned exponent[R];
            const int b = c / kR8Block, word = (b >> 2) * 512 + (b & 3);
#pragma unroll
            for (int u = 0; u < R; ++u) {
                code[u] = make_uint2(0u, 0u);
                exponent[u] = 255u;                                 // a row that is not there is NaN
                if (src[u]) {
                    if (E == 8) code[u] = __ldg(reinterpret_cast<const uint2*>(src[u] + c));
                    else if (E == 4) code[u].x = __ldg(reinterpret_cast<const unsigned*>(src[u] + c));
                    else if (E == 2) code[u].x = __ldg(reinterpret_cast<const unsigned short*>(src[u] + c));
                    else code[u].x = __ldg(src[u] + c);
                    exponent[u] = __ldg(sf[u] + word);
                }
            }
#pragma unroll
            for (int u = 0; u < R; ++u) {
                const int64_t i = first + u * groups;
                if (i >= m) break;
                const float scale = r8_scale_value(exponent[u]);
                T* dst = out + i * ld + c;
                const unsigned w[2] = {code[u].x, code[u].y};
                __align__(16) T o[E < 2 ? 2 : E];
#pragma unroll
                for (int k = 0; k < E; k += 2) {
                    const float2 v = from_e4m3x2(w[k >> 2] >> (8 * (k & 2)) & 0xffffu);
                    r8_narrow(o[k], mul_keep(v.x, scale));
                    r8_narrow(o[k + 1], mul_keep(v.y, scale));
                }
                constexpr int kBytes = E * (int)sizeof(T);
                if (kBytes == 16) __stcs(reinterpret_cast<uint4*>(dst), *reinterpret_cast<const uint4*>(o));
                else if (kBytes == 8) __stcs(reinterpret_cast<uint2*>(dst), *reinterpret_cast<const uint2*>(o));
                else if (E > 1) __stcs(reinterpret_cast<unsigned*>(dst), *reinterpret_cast<const unsigned*>(o));
                else dst[0] = o[0];
            }
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
