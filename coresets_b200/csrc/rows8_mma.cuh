// Rows in 8 bits: products of the rows of two stores on the tensor cores, with the epilogues that use
// them (the product itself; the distance of every row to the nearest centre).  This file: few columns
// (at most 64), which all stand in one tile; rows8_pair.cuh: many.
// Part of the single translation unit fps_kernels.cu (included there, in order).
//
//   P[i, j] = sum over blocks b of 128 of 2^(ea[i,b] + eb[j,b]) * sum over the block of a_i * b_j
//
// Powers of two are scales that tcgen05.mma kind::mxf8f6f4 applies by itself (one exponent byte per 32
// elements of a row; the four quarters of a block of 128 name the same byte), so the whole sum over D
// accumulates in TMEM in float32 and nothing has to be promoted between blocks.  Measured: a step takes its 32 terms
// and the accumulator, cuts each off at 2^-25 of the largest one's power of two, and cuts the sum off toward zero to 24
// bits.  That is the choice of rounding here; sums of one sign lose 1.8e-7 at D = 1024, 1.5e-6 at 4096, 6e-5 at 65536.
//
// One block per SM: warp 0 copies (TMA, 128-byte swizzle; the exponents stand in the store in the
// order that tcgen05.cp wants, 512 bytes per 128 rows and 4 blocks), warp 1 issues the MMAs, the other
// warps read the accumulators back.  Rows of the "lane" operand are the 128 TMEM lanes of a tile, rows
// of the "column" operand its NT columns.  Every wait is bounded; one that runs out sets the store's
// status word and the whole block drains and leaves.
#ifndef CORESETS_B200_ROWS8_MMA_CUH
#define CORESETS_B200_ROWS8_MMA_CUH

namespace {

enum { R8_PRODUCTS = 0, R8_COVERAGE = 1 };
constexpr int kR8Lanes = 128;                       // rows of the lane operand in a tile
// The bound of every wait, that of the engine's pipes; short where a test makes one run out.
constexpr unsigned long long kR8WaitNs = 10000000000ull, kR8TestWaitNs = 20000000ull;

struct R8Job {
    const unsigned char* lane_scales;
    const unsigned char* col_scales;
    const float* lane_norms;                        // coverage only
    const float* col_norms;
    int64_t n_lane, n_col;                          // rows of the two operands
    int D, words;
    int width;                                      // bytes of a row in a tile: 16, 32, 64 or 128 (a block of 128, or the whole row)
    int col_tiles;                                  // rows8_pair.cuh: column tiles, and tiles in all
    int64_t tiles;
    int64_t items;                                  // here: lane tiles (one tile holds all columns)
    void* out;                                      // products: P; coverage: h
    int64_t lane_stride, col_stride;                // products, in elements
    int bulk_out;                                   // products: out takes bulk stores
    int keep;                                       // coverage: min with what h holds
    int* status;
    int stall;                                      // test hook: the producer starts no copy, so that the waits run out
    unsigned long long wait_ns;
};

__device__ __forceinline__ uint64_t umma_desc(const uint32_t smem, const uint32_t stride_bytes, const uint64_t swizzle) {
    // start >> 4, stride between the 16-byte halves of a step's codes >> 4 (1; unused with a swizzle), stride
    // between groups of 8 rows >> 4, the constant 1 of this architecture, swizzle mode
    return (uint64_t)((smem & 0x3ffffu) >> 4) | (1ull << 16) | ((uint64_t)(stride_bytes >> 4) << 32) | (1ull << 46) | (swizzle << 61);
}
// Codes of a tile: rows of `width` bytes, swizzled over that width (16: not swizzled, and the step's second 16 codes are
// `lbo` bytes further on, where the tile holds zeros).
__device__ __forceinline__ uint64_t tile_desc(const uint32_t smem, const int width, const uint32_t lbo) {
    const uint64_t d = umma_desc(smem, 8u * (uint32_t)width, width == 128 ? 2u : (width == 64 ? 4u : (width == 32 ? 6u : 0u)));
    return width == 16 ? d + ((uint64_t)((lbo >> 4) - 1u) << 16) : d;
}
__device__ __forceinline__ void zero_smem(unsigned char* p, const int bytes) {
    for (int i = 16 * (int)threadIdx.x; i < bytes; i += 16 * (int)blockDim.x) *reinterpret_cast<uint4*>(p + i) = make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, const int x, const int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
// rows of 16 bytes are one sequence in memory and in the tile: x in units of 8 bytes
__device__ __forceinline__ void tma_line(void* dst, const CUtensorMap* map, const int x, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.1d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2}], [%3];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(smem_u32(bar)) : "memory");
}
// One bulk store, from shared memory, of a box of the map's; what of it lies past the last row or column is left out.
// Results are marked as the first to leave L2, for the operands' sake (4096 x 100 000 x 128 to bfloat16: 192 -> 172 us,
// 20 000 x 20 000 x 128 to float32: 362 -> 343).
__device__ __forceinline__ void r8_store_tile(const CUtensorMap* map, const int x, const int y, const uint32_t smem) {
    unsigned long long policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group.L2::cache_hint [%0, {%1, %2}], [%3], %4;"
                 ::"l"(map), "r"(x), "r"(y), "r"(smem), "l"(policy) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// one element of a result, likewise
__device__ __forceinline__ void r8_put(float* p, const float v) { __stcs(p, v); }
template <typename T>
__device__ __forceinline__ void r8_put(T* p, const T v) {
    __stcs(reinterpret_cast<unsigned short*>(p), *reinterpret_cast<const unsigned short*>(&v));
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_copy_scales(const uint32_t tmem, const uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void tc_mma(const uint32_t acc, const uint64_t a, const uint64_t b, const uint32_t idesc,
                                       const uint32_t sfa, const uint32_t sfb, const bool add) {
    asm volatile("{ .reg .pred p; setp.ne.u32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p; }"
                 ::"r"(acc), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((unsigned)add) : "memory");
}
__device__ __forceinline__ void tc_load(const uint32_t tmem, unsigned (&u)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
                   "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]),
                   "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]),
                   "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
                 : "r"(tmem) : "memory");
}
__device__ __forceinline__ void tc_load(const uint32_t tmem, unsigned (&u)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
                   "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
                 : "r"(tmem) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// One lane of a converged warp.  The copy and MMA instructions take their descriptors from uniform
// registers: under a branch that the compiler cannot see to be one lane's each of them costs ~230 clocks
// (products 8192^3: 968 us that way), so the warps' loops run converged and only the issue is elected.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p != 0;
}

// Wait that also ends when another role has given up.  The clock is looked at only after a number of tries
// (each of which the hardware may itself hold for a while).
struct R8Bound {
    volatile int* abort_flag;
    unsigned long long ns;
};
__device__ __forceinline__ bool r8_wait(uint64_t* b, const uint32_t parity, const R8Bound& bound) {
    if (mbar_try(b, parity)) return true;
    unsigned long long t0 = 0;
    for (;;) {
#pragma unroll 1
        for (int it = 0; it < 64; ++it)
            if (mbar_try(b, parity)) return true;
        if (*bound.abort_flag) return false;
        const unsigned long long now = global_ns();
        if (t0 == 0) t0 = now;
        if (now - t0 > bound.ns) {
            *bound.abort_flag = 1;
            return false;
        }
    }
}

// the same by a whole converged warp
__device__ __forceinline__ bool r8_wait_warp(uint64_t* b, const uint32_t parity, const R8Bound& bound) {
    return __all_sync(kFull, r8_wait(b, parity, bound));
}

template <int NT, int WHAT, typename T> struct R8Shape {
    static constexpr int kTileA = kR8Lanes * kR8Block, kTileB = NT * kR8Block;
    static constexpr int kStage = kTileA + kTileB + 1024;              // two tiles, two scale words of 128 rows
    static constexpr int kAcc = 256 / (NT < 32 ? 32 : NT);             // accumulators: 8, 8, 4; the way from a tile's last MMA to its
                                                                       // free accumulator is much longer than its few MMAs
    // Sets of four reading warps (a set has the tile's 128 lanes), tile by tile in turn: a reader's way from accumulator to
    // memory is long, and what a tile takes else is short (461k x 10 x 16 to float16: 39 us with one set, 34 with four;
    // 1M x 64 x 128: coverage 49 -> 33).  kAcc is a multiple of it, so that the wait for an accumulator's fill comes after the
    // same set's wait for the fill before.
    static constexpr int kSets = kAcc / 2;
    static constexpr int kThreads = 64 + 128 * kSets;
    // a reader's products on their way out
    static constexpr int kOutWarp = WHAT == R8_PRODUCTS ? (32 * (NT + 1) * (int)sizeof(T) + 127) & ~127 : 0;
    static constexpr int kOut = 4 * kSets * kOutWarp;
    static constexpr int kFit = (226 * 1024 - kOut - 1024 - 2048) / kStage;
    static constexpr int kStages = kFit < 8 ? kFit : 8;
    static constexpr int kSmem = kStages * kStage + kOut + 1024;       // slack to align the tiles to 1 KB
};

// NARROW: rows of at most 64 codes (one step or two of the MMA), tiles of job.width bytes a row.
template <int NT, int WHAT, typename T, bool NARROW>
__global__ void __launch_bounds__((R8Shape<NT, WHAT, T>::kThreads), 1) rows8_mma_kernel(const __grid_constant__ CUtensorMap lane_map,
                                                           const __grid_constant__ CUtensorMap col_map,
                                                           const __grid_constant__ CUtensorMap out_map, const R8Job job) {
    using S = R8Shape<NT, WHAT, T>;
    constexpr int NC = NT < 32 ? NT : 32;                              // columns read back at a time
    extern __shared__ unsigned char s_raw[];
    __shared__ uint64_t s_full[S::kStages], s_empty[S::kStages], s_acc_full[S::kAcc], s_acc_empty[S::kAcc];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort_word;
    __shared__ __align__(16) float s_norm[4 * S::kSets][NT < 32 ? 32 : NT];          // a copy per reading warp: no barrier between them
    const R8Bound s_abort{&s_abort_word, job.wait_ns};
    unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)s_raw + 1023) & ~(uintptr_t)1023);

    const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;    // warp: known to be uniform
    const int kblocks = (job.D + kR8Block - 1) / kR8Block;
    if (threadIdx.x == 0) {
        s_abort_word = 0;
        for (int i = 0; i < S::kStages; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], 1); }
        for (int i = 0; i < S::kAcc; ++i) { mbar_init(&s_acc_full[i], 1); mbar_init(&s_acc_empty[i], 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const int width = NARROW ? job.width : kR8Block;
    if (NARROW && width == 16) {
        for (int i = 0; i < S::kStages; ++i) {
            zero_smem(tiles + i * S::kStage + kR8Lanes * 64, kR8Lanes * 16);
            zero_smem(tiles + i * S::kStage + S::kTileA + NT * 64, NT * 16);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(kFull, s_tmem, 0);
    constexpr uint32_t kSf = 256;                                      // scale columns: 4 + 4 per stage behind the accumulators

    if (warp == 0) {
        uint32_t n = 0;                                                // stages filled so far
        bool ok = !job.stall;
        for (int64_t item = blockIdx.x; item < job.items && ok; item += gridDim.x) {
            for (int kb = 0; kb < kblocks; ++kb, ++n) {
                const uint32_t st = n % S::kStages, round = n / S::kStages;
                if (round > 0 && !r8_wait_warp(&s_empty[st], (round - 1) & 1u, s_abort)) { ok = false; break; }
                unsigned char* a = tiles + st * S::kStage;
                if (elect_one()) {
                    mbar_expect_tx(&s_full[st], (uint32_t)((kR8Lanes + NT) * width + 1024));
                    if (NARROW && width == 16) {
                        tma_line(a, &lane_map, (int)(item * kR8Lanes * 2), &s_full[st]);
                        tma_line(a + S::kTileA, &col_map, 0, &s_full[st]);
                    } else {
                        tma_tile(a, &lane_map, kb * kR8Block, (int)(item * kR8Lanes), &s_full[st]);
                        tma_tile(a + S::kTileA, &col_map, kb * kR8Block, 0, &s_full[st]);
                    }
                    bulk_load(a + S::kTileA + S::kTileB, job.lane_scales + (item * job.words + (kb >> 2)) * 512, 512, &s_full[st]);
                    bulk_load(a + S::kTileA + S::kTileB + 512, job.col_scales + (kb >> 2) * 512, 512, &s_full[st]);
                }
                __syncwarp();
            }
        }
        // the last releases of the stages have arrived before the block leaves
        for (uint32_t k = n > S::kStages ? n - S::kStages : 0; k < n && ok; ++k)
            ok = r8_wait_warp(&s_empty[k % S::kStages], (k / S::kStages) & 1u, s_abort);
        // no copy may be in flight when the block leaves: the last fills of every stage (already
        // complete unless a consumer gave up)
        if (!ok)
            for (uint32_t k = n > S::kStages ? n - S::kStages : 0; k < n; ++k)
                for (int it = 0; it < (1 << 16) && !mbar_try(&s_full[k % S::kStages], (k / S::kStages) & 1u); ++it) {}
    } else if (warp == 1) {
        uint32_t n = 0, t = 0;
        bool ok = true;
        // e4m3 x e4m3, K-major, float32 accumulators, exponent-only scales, M = 128
        constexpr uint32_t kIdesc = ((uint32_t)(NT >> 3) << 17) | (1u << 23) | ((uint32_t)(kR8Lanes >> 4) << 24);
        for (int64_t item = blockIdx.x; item < job.items && ok; item += gridDim.x, ++t) {
            const uint32_t buf = t % S::kAcc, round = t / S::kAcc;
            if (round > 0 && !r8_wait_warp(&s_acc_empty[buf], (round - 1) & 1u, s_abort)) { ok = false; break; }
            tc_fence_after();
            const uint32_t acc = tmem + buf * (256 / S::kAcc);
            for (int kb = 0; kb < kblocks; ++kb, ++n) {
                const uint32_t st = n % S::kStages;
                if (!r8_wait_warp(&s_full[st], (n / S::kStages) & 1u, s_abort)) { ok = false; break; }
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t a = smem_u32(tiles + st * S::kStage), b = a + S::kTileA, sf = b + S::kTileB;
                    const uint32_t sfa = tmem + kSf + st * 8, sfb = sfa + 4;
                    tc_copy_scales(sfa, umma_desc(sf, 128, 0));
                    tc_copy_scales(sfb, umma_desc(sf + 512, 128, 0));
                    const uint32_t id = kIdesc | ((uint32_t)(kb & 3) << 4) | ((uint32_t)(kb & 3) << 29);
                    const int left = job.D - kb * kR8Block, steps = left >= kR8Block ? 4 : (left + 31) >> 5;
                    if constexpr (!NARROW) {
                        const uint64_t da = umma_desc(a, 1024, 2), db = umma_desc(b, 1024, 2);
                        for (int k = 0; k < steps; ++k) tc_mma(acc, da + 2 * k, db + 2 * k, id, sfa, sfb, kb > 0 || k > 0);
                    } else {
                        const uint64_t da = tile_desc(a, width, kR8Lanes * 64), db = tile_desc(b, width, NT * 64);
                        for (int k = 0; k < steps; ++k) tc_mma(acc, da + 2 * k, db + 2 * k, id, sfa, sfb, k > 0);
                    }
                    tc_commit(&s_empty[st]);
                    if (kb == kblocks - 1) tc_commit(&s_acc_full[buf]);
                }
                __syncwarp();
            }
        }
        // the tensor core may still read the stages of a drained block: wait for what was issued
        if (!ok)
            for (uint32_t k = n > S::kStages ? n - S::kStages : 0; k < n; ++k)
                for (int it = 0; it < (1 << 16) && !mbar_try(&s_empty[k % S::kStages], (k / S::kStages) & 1u); ++it) {}
    } else {
        const int quad = warp & 3, set = (warp - 2) >> 2, reader = warp - 2;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        uint32_t t = 0;
        bool ok = true;
        if (WHAT == R8_COVERAGE) {
            // the centres' norms; a column past the last centre can never be the nearest
            for (int c = lane; c < NT; c += 32) s_norm[reader][c] = c < job.n_col ? __ldg(job.col_norms + c) : __uint_as_float(0x7f800000u);
            __syncwarp();
        }
        for (int64_t item = blockIdx.x; item < job.items && ok; item += gridDim.x, ++t) {
            if (t % S::kSets != (uint32_t)set) continue;
            const int64_t row = item * kR8Lanes + quad * 32 + lane;
            const uint32_t buf = t % S::kAcc;
            float row_norm = 0.0f, had = __uint_as_float(0x7f800000u);      // (ahead of the wait)
            if (WHAT == R8_COVERAGE && row < job.n_lane) {
                row_norm = __ldg(job.lane_norms + row);
                if (job.keep) had = reinterpret_cast<const float*>(job.out)[row];
            }
            ok = r8_wait_warp(&s_acc_full[buf], (t / S::kAcc) & 1u, s_abort);
            if (!ok) break;
            tc_fence_after();
            unsigned v[NT];
#pragma unroll
            for (int c = 0; c < NT; c += NC) tc_load(lanes + buf * (256 / S::kAcc) + c, *reinterpret_cast<unsigned(*)[NC]>(v + c));
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_acc_empty[buf]);
            if (WHAT == R8_PRODUCTS) {
                T* mine = reinterpret_cast<T*>(tiles + S::kStages * S::kStage + reader * S::kOutWarp);
                if (job.bulk_out) {
                    // NT columns x 32 lanes through shared memory, one bulk store for the warp
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < NT; ++j) r8_narrow(mine[j * 32 + lane], __uint_as_float(v[j]));
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0 && row < job.n_lane) r8_store_tile(&out_map, (int)row, 0, smem_u32(mine));
                } else if (job.col_stride == 1) {
                    // the rows of `out` follow the columns: 32 rows of n_col elements through shared memory, stored in
                    // their order (1M x 64 x 128 to float32: 139 us, each lane storing its own row 360)
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < NT; ++j) r8_narrow(mine[lane * (NT + 1) + j], __uint_as_float(v[j]));
                    __syncwarp();
                    const int n_col = (int)job.n_col, rows = (int)(job.n_lane - (row - lane) < 32 ? job.n_lane - (row - lane) : 32);
                    const unsigned inverse = n_col > 1 ? (unsigned)((0x100000000ull + n_col - 1) / n_col) : 0u;
                    T* out = reinterpret_cast<T*>(job.out) + (row - lane) * job.lane_stride;
                    const int last = rows * n_col;
#pragma unroll 1
                    for (int e0 = lane; e0 < last; e0 += 8 * 32) {
                        T o[8];
                        int64_t at[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            const int e = e0 + 32 * u < last ? e0 + 32 * u : last - 1;      // (past the end: its last element again)
                            const int r = n_col > 1 ? (int)__umulhi((unsigned)e, inverse) : e, c = e - r * n_col;
                            o[u] = mine[r * (NT + 1) + c];
                            at[u] = r * job.lane_stride + c;
                        }
#pragma unroll
                        for (int u = 0; u < 8; ++u) r8_put(out + at[u], o[u]);
                    }
                } else if (row < job.n_lane) {
                    T* out = reinterpret_cast<T*>(job.out) + row * job.lane_stride;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        if (j < job.n_col) {
                            T o;
                            r8_narrow(o, __uint_as_float(v[j]));
                            r8_put(out + j * job.col_stride, o);
                        }
                }
            } else if (row < job.n_lane) {
                // |a - c|^2 = |a|^2 + (|c|^2 - 2 a.c); a NaN never lowers h, rounding never makes it negative
                float best[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) best[j] = __uint_as_float(0x7f800000u);
#pragma unroll
                for (int j = 0; j < NT; ++j) best[j & 3] = fminf(best[j & 3], __fmaf_rn(-2.0f, __uint_as_float(v[j]), s_norm[reader][j]));
                const float d = __fadd_rn(row_norm, fminf(fminf(best[0], best[1]), fminf(best[2], best[3])));
                const float up = d == d ? fmaxf(d, 0.0f) : __uint_as_float(0x7f800000u);
                float* h = reinterpret_cast<float*>(job.out) + row;
                *h = up < had ? up : had;               // (a NaN there stays)
            }
        }
        if (WHAT == R8_PRODUCTS && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0 && s_abort_word && job.status) *job.status = ST_PIPE_TIMEOUT;
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

__global__ void rows8_fill_kernel(float* h, const int64_t n, const float v) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) h[i] = v;
}

}  // namespace

#endif  // CORESETS_B200_ROWS8_MMA_CUH
