// Rows in 8 bits: the products of rows8_mma.cuh for many columns, on pairs of SMs.
// Part of the single translation unit fps_kernels.cu (included there, in order).
//
// A cluster of two blocks works on one tile of 256 lanes x 192 columns (tcgen05 cta_group::2): each block
// holds 128 rows of the lane operand and half of the column operand's rows, and each tensor core reads the
// halves of both.  That halves what a block has to fetch for its share of the column operand.  TMEM: two
// accumulators of 192 columns, and per stage 4 + 8 columns of scales.
// The even block ("leader") issues every MMA; the full and the accumulator-free barriers are its own,
// the stage-free and the accumulator-full barriers exist in both blocks and are reached by multicast commits.
#ifndef CORESETS_B200_ROWS8_PAIR_CUH
#define CORESETS_B200_ROWS8_PAIR_CUH

namespace {

constexpr int kPairCols = 192, kPairLanes = 256;
constexpr int kPairStages = 7, kPairReaders = 16, kPairWarps = 2 + kPairReaders;
constexpr int kPairPart = kPairCols / (kPairReaders / 4);        // columns of a reading warp
constexpr int kPairSlots = 8;                                   // TMEM slots of scales, one per 4 blocks of a row: a slot comes round
                                                                // after 8 stages at least, when the stage 7 back is known to be done
constexpr int kPairA = kR8Lanes * kR8Block, kPairB = kPairCols / 2 * kR8Block;
constexpr int kPairSf = 512 + 1024;                              // scale words of 128 lanes, and of the columns' two chunks of 128
constexpr int kPairStage = (kPairA + kPairB + kPairSf + 1023) & ~1023;
constexpr int kPairSmem = kPairStages * kPairStage + 1024;

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the same shared-memory object in the leader's block
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}
__device__ __forceinline__ void pair_tile(const uint32_t dst, const CUtensorMap* map, const int x, const int y, const uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void pair_scales(const uint32_t dst, const CUtensorMap* map, const int w, const int chunk, const uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(0), "r"(w), "r"(chunk), "r"(bar) : "memory");
}
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((unsigned short)3) : "memory");
}
__device__ __forceinline__ void pair_copy_scales(const uint32_t tmem, const uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void pair_mma(const uint32_t acc, const uint64_t a, const uint64_t b, const uint32_t idesc,
                                         const uint32_t sfa, const uint32_t sfb, const bool add) {
    asm volatile("{ .reg .pred p; setp.ne.u32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p; }"
                 ::"r"(acc), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((unsigned)add) : "memory");
}
// two at a time: (a, b) * (s, s) + (c, d)
__device__ __forceinline__ float2 fma2(const float a, const float b, const float s, const float2 c) {
    float2 r;
    asm("{ .reg .b64 x, y, z;\n mov.b64 x, {%2, %3}; mov.b64 y, {%4, %4}; mov.b64 z, {%5, %6};\n"
        "fma.rn.ftz.f32x2 x, x, y, z; mov.b64 {%0, %1}, x; }"
        : "=f"(r.x), "=f"(r.y) : "f"(a), "f"(b), "f"(s), "f"(c.x), "f"(c.y));
    return r;
}

__device__ __forceinline__ float min3(const float a, const float b, const float c) {
    float r;
    asm("min.ftz.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 48 columns at once: both loads in flight before the wait
__device__ __forceinline__ void tc_load48(const uint32_t tmem, unsigned (&u)[48]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%48];\n"
                 "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47}, [%49];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
                   "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]),
                   "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]),
                   "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31]),
                   "=r"(u[32]), "=r"(u[33]), "=r"(u[34]), "=r"(u[35]), "=r"(u[36]), "=r"(u[37]), "=r"(u[38]), "=r"(u[39]),
                   "=r"(u[40]), "=r"(u[41]), "=r"(u[42]), "=r"(u[43]), "=r"(u[44]), "=r"(u[45]), "=r"(u[46]), "=r"(u[47])
                 : "r"(tmem), "r"(tmem + 32) : "memory");
}

struct PairSpan { int64_t lt; int c0, c1; };
__device__ __forceinline__ PairSpan pair_span(const R8Job& job, const int64_t item) {
    PairSpan s;
    s.lt = item / job.splits;
    s.c0 = (int)(item % job.splits) * job.col_split;
    s.c1 = s.c0 + job.col_split < job.col_tiles ? s.c0 + job.col_split : job.col_tiles;
    return s;
}

template <int WHAT, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairWarps * 32, 1)
rows8_pair_kernel(const __grid_constant__ CUtensorMap lane_map, const __grid_constant__ CUtensorMap col_map,
                  const __grid_constant__ CUtensorMap lane_sf_map, const __grid_constant__ CUtensorMap col_sf_map, const R8Job job) {
    extern __shared__ unsigned char s_raw[];
    __shared__ uint64_t s_full[kPairStages], s_empty[kPairStages], s_acc_full[2], s_acc_empty[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort_word;
    __shared__ __align__(16) float s_norm[kPairReaders][kPairPart];
    volatile int* s_abort = &s_abort_word;
    unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)s_raw + 1023) & ~(uintptr_t)1023);

    const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;    // warp: known to be uniform
    const uint32_t rank = cluster_rank();
    const int64_t first = blockIdx.x >> 1, stride = gridDim.x >> 1;
    const int kblocks = (job.D + kR8Block - 1) / kR8Block;
    if (threadIdx.x == 0) {
        s_abort_word = 0;
        for (int i = 0; i < kPairStages; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&s_acc_full[i], 1); mbar_init(&s_acc_empty[i], 2 * kPairReaders); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(kFull, s_tmem, 0);
    constexpr uint32_t kSf = 2 * kPairCols;

    if (warp == 0) {
        uint32_t st = 0, phase = 0;
        uint32_t n = 0;
        bool ok = true;
        for (int64_t item = first; item < job.items && ok; item += stride) {
            const PairSpan sp = pair_span(job, item);
            const int row = (int)(sp.lt * kPairLanes) + (int)rank * kR8Lanes;
            for (int ct = sp.c0; ct < sp.c1 && ok; ++ct)
                for (int kb = 0; kb < kblocks; ++kb, ++n) {
                    if (n >= kPairStages && !r8_wait_warp(&s_empty[st], phase ^ 1u, s_abort)) { ok = false; break; }
                    const uint32_t a = smem_u32(tiles + st * kPairStage), bar = leader_addr(&s_full[st]);
                    const bool scales = (kb & 3) == 0;
                    if (elect_one()) {
                        if (rank == 0) mbar_expect_tx(&s_full[st], 2 * (kPairA + kPairB + (scales ? kPairSf : 0)));
                        pair_tile(a, &lane_map, kb * kR8Block, row, bar);
                        pair_tile(a + kPairA, &col_map, kb * kR8Block, ct * kPairCols + (int)rank * (kPairCols / 2), bar);
                        if (scales) {
                            pair_scales(a + kPairA + kPairB, &lane_sf_map, kb >> 2, row >> 7, bar);
                            pair_scales(a + kPairA + kPairB + 512, &col_sf_map, kb >> 2, ct * kPairCols >> 7, bar);
                        }
                    }
                    __syncwarp();
                    if (++st == kPairStages) { st = 0; phase ^= 1u; }
                }
        }
        // no copy may be in flight when the pair leaves (they all are complete unless a role gave up)
        if (!ok && rank == 0)
            for (uint32_t k = n > kPairStages ? n - kPairStages : 0; k < n; ++k)
                for (int it = 0; it < (1 << 16) && !mbar_try(&s_full[k % kPairStages], (k / kPairStages) & 1u); ++it) {}
    } else if (warp == 1) {
        if (rank == 0) {
            uint32_t st = 0, phase = 0, slot = 0;
            uint32_t n = 0, t = 0;
            bool ok = true;
            constexpr uint32_t kIdesc = ((uint32_t)(kPairCols >> 3) << 17) | (1u << 23) | ((uint32_t)(kPairLanes >> 4) << 24);
            const uint32_t base = smem_u32(tiles);
            for (int64_t item = first; item < job.items && ok; item += stride) {
                const PairSpan sp = pair_span(job, item);
                for (int ct = sp.c0; ct < sp.c1 && ok; ++ct, ++t) {
                    const uint32_t buf = t & 1u, round = t >> 1;
                    if (round > 0 && !r8_wait_warp(&s_acc_empty[buf], (round - 1) & 1u, s_abort)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t acc = tmem + buf * kPairCols;
                    // the tile's first column within its chunk of 128 scales: 32 rows a TMEM column
                    const uint32_t sub = (uint32_t)(ct * kPairCols & 127) >> 5;
                    for (int kb = 0; kb < kblocks; ++kb, ++n) {
                        if (!r8_wait_warp(&s_full[st], phase, s_abort)) { ok = false; break; }
                        tc_fence_after();
                        if ((kb & 3) == 0 && ++slot == kPairSlots) slot = 0;
                        if (elect_one()) {
                            const uint32_t a = base + st * kPairStage, b = a + kPairA, sf = b + kPairB;
                            const uint32_t sfa = tmem + kSf + slot * 12, sfb = sfa + 4;
                            if ((kb & 3) == 0) {
                                pair_copy_scales(sfa, umma_desc(sf, 128, 0));
                                pair_copy_scales(sfb, umma_desc(sf + 512, 128, 0));
                                pair_copy_scales(sfb + 4, umma_desc(sf + 1024, 128, 0));
                            }
                            const uint32_t id = kIdesc | ((uint32_t)(kb & 3) << 4) | ((uint32_t)(kb & 3) << 29);
                            const int left = job.D - kb * kR8Block;
                            const uint64_t da = umma_desc(a, 1024, 2), db = umma_desc(b, 1024, 2);
                            if (left > 96) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) pair_mma(acc, da + 2 * k, db + 2 * k, id, sfa, sfb + sub, kb > 0 || k > 0);
                            } else {
                                const int steps = (left + 31) >> 5;
                                for (int k = 0; k < steps; ++k) pair_mma(acc, da + 2 * k, db + 2 * k, id, sfa, sfb + sub, kb > 0 || k > 0);
                            }
                            pair_commit(&s_empty[st]);
                            if (kb == kblocks - 1) pair_commit(&s_acc_full[buf]);
                        }
                        __syncwarp();
                        if (++st == kPairStages) { st = 0; phase ^= 1u; }
                    }
                }
            }
            if (!ok)
                for (uint32_t k = n > kPairStages ? n - kPairStages : 0; k < n; ++k)
                    for (int it = 0; it < (1 << 16) && !mbar_try(&s_empty[k % kPairStages], (k / kPairStages) & 1u); ++it) {}
        }
    } else {
        const int quad = warp & 3, part = (warp - 2) >> 2;
        float* norm = s_norm[warp - 2];
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16) + part * kPairPart;
        const float inf = __uint_as_float(0x7f800000u);
        uint32_t t = 0;
        bool ok = true;
        for (int64_t item = first; item < job.items && ok; item += stride) {
            const PairSpan sp = pair_span(job, item);
            const int64_t row = sp.lt * kPairLanes + rank * kR8Lanes + quad * 32 + lane;
            float best[4] = {inf, inf, inf, inf};
            // the centres' norms of the next tile, one tile ahead; past the last centre nothing is near
            float2 ahead;
            const auto fetch = [&](const int ct) {
                const int64_t col = (int64_t)ct * kPairCols + part * kPairPart + 2 * lane;
                ahead.x = 2 * lane < kPairPart && col < job.n_col ? __ldg(job.col_norms + col) : inf;
                ahead.y = 2 * lane < kPairPart && col + 1 < job.n_col ? __ldg(job.col_norms + col + 1) : inf;
            };
            if (WHAT == R8_COVERAGE) fetch(sp.c0);
            for (int ct = sp.c0; ct < sp.c1 && ok; ++ct, ++t) {
                const uint32_t buf = t & 1u;
                if (WHAT == R8_COVERAGE) {
                    __syncwarp();
                    if (2 * lane < kPairPart) *reinterpret_cast<float2*>(norm + 2 * lane) = ahead;
                    __syncwarp();
                    if (ct + 1 < sp.c1) fetch(ct + 1);
                }
                ok = r8_wait_warp(&s_acc_full[buf], (t >> 1) & 1u, s_abort);
                if (!ok) break;
                tc_fence_after();
                unsigned v[kPairPart];
                tc_load48(lanes + buf * kPairCols, v);
                // the accumulator is free as soon as it is in registers.  (A plain arrive: one with a release
                // over the cluster waits for all of the warp's memory, 600 clocks a tile.)
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(&s_acc_empty[buf])) : "memory");
                if (WHAT == R8_PRODUCTS) {
                    const int64_t col = (int64_t)ct * kPairCols + part * kPairPart;
                    T* out = reinterpret_cast<T*>(job.out) + row * job.lane_stride + col * job.col_stride;
                    if (row < job.n_lane) {
#pragma unroll
                        for (int j = 0; j < kPairPart; ++j)
                            if (col + j < job.n_col) {
                                T o;
                                r8_narrow(o, __uint_as_float(v[j]));
                                out[j * job.col_stride] = o;
                            }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kPairPart; j += 4) {
                        const float4 n4 = *reinterpret_cast<const float4*>(norm + j);
                        const float2 p = fma2(__uint_as_float(v[j]), __uint_as_float(v[j + 1]), -2.0f, make_float2(n4.x, n4.y));
                        const float2 q = fma2(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]), -2.0f, make_float2(n4.z, n4.w));
                        best[(j >> 1) & 3] = min3(best[(j >> 1) & 3], p.x, p.y);
                        best[((j >> 1) + 1) & 3] = min3(best[((j >> 1) + 1) & 3], q.x, q.y);
                    }
                }
            }
            if (WHAT == R8_COVERAGE && ok && row < job.n_lane) {
                const float d = __fadd_rn(__ldg(job.lane_norms + row), fminf(fminf(best[0], best[1]), fminf(best[2], best[3])));
                if (d == d)      // h holds +inf or what it had: a NaN leaves that; max(d, 0) orders like its bits
                    atomicMin(reinterpret_cast<int*>(job.out) + row, __float_as_int(fmaxf(d, 0.0f)));
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    if (threadIdx.x == 0 && s_abort_word && job.status) *job.status = ST_PIPE_TIMEOUT;
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace

#endif  // CORESETS_B200_ROWS8_PAIR_CUH
