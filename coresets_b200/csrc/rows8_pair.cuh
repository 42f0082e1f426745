// Rows in 8 bits: the products of rows8_mma.cuh for many columns, on pairs of SMs.
// Part of the single translation unit fps_kernels.cu (included there, in order).
//
// A cluster of two blocks works on one tile of 256 lanes x 192 columns (tcgen05 cta_group::2): each block
// holds 128 rows of the lane operand and half of the column operand's rows, and each tensor core reads the
// halves of both.  That halves what a block has to fetch for its share of the column operand.  TMEM: two
// accumulators of 192 columns, and per stage 4 + 8 columns of scales.
//
// Coverage needs max_j (a.c_j - |c_j|^2 / 2) per row.  The norms come in through the tensor core as one more
// step of 32 elements: -|c|^2 / 2 is a 24-bit number, six digits of 4 bits that e4m3 holds exactly, times
// six powers of two that stand in the lane operand, times one exponent per column.  The readers are left with one
// three-input maximum per two columns.  Reading the norms from shared memory instead costs 4 wavefronts per
// 16 bytes, and that pipe then sets the pace (1M x 128 by 8192 centres: 1.28 ms; with the extra step 1.10 ms).
//
// The even block ("leader") issues every MMA; the full and the accumulator-free barriers are its own,
// the stage-free and the accumulator-full barriers exist in both blocks and are reached by multicast commits.
#ifndef CORESETS_B200_ROWS8_PAIR_CUH
#define CORESETS_B200_ROWS8_PAIR_CUH

namespace {

constexpr int kPairCols = 192, kPairLanes = 256;
constexpr int kPairReaders = 16, kPairWarps = 3 + kPairReaders;
constexpr int kPairPart = kPairCols / (kPairReaders / 4);        // columns of a reading warp
constexpr int kPairA = kR8Lanes * kR8Block, kPairB = kPairCols / 2 * kR8Block;
constexpr int kPairSf = 512 + 1024;                              // scale words of 128 lanes, and of the columns' two chunks of 128
constexpr int kPairNormB = kPairCols / 2 * 16, kPairNormSf = 1024;          // digits of the norms, and their exponents
// KEEP: the lane operand of a segment (128 rows of at most 8 blocks, two segments where they have at most 4) stays in shared
// memory while its column tiles pass, instead of coming in with every stage.  The MMAs take as many clocks as before,
// but the SMs draw less power and clock higher: 500k x 256 by 10 000 centres 1073 -> 1024 us, 300k x 1024 by 8192 1720 -> 1615.
constexpr int kPairKept = 8;
template <int WHAT, typename T, bool KEEP> struct PairShape {
    static constexpr bool kNorms = WHAT == R8_COVERAGE;
    static constexpr int kOut = kNorms ? 0 : kPairReaders * kPairPart * 32 * (int)sizeof(T);     // a reading warp's share of a tile of products
    static constexpr int kStages = KEEP ? 5 : (!kNorms && sizeof(T) == 4 ? 4 : 6);
    static constexpr int kTile = (KEEP ? 0 : kPairA) + kPairB;                 // codes of a stage
    static constexpr int kKept = KEEP ? kPairKept * kPairA : 0;                // lane operand of whole segments
    // what else a stage may bring in (digits end with 16 zero bytes)
    static constexpr int kFirst = (kPairSf + (kNorms ? kPairNormSf + kPairNormB + 16 : 0) + 127) & ~127;
    static constexpr int kSmem = kKept + kStages * (kTile + kFirst) + kOut + 1024;
    // TMEM columns of scales, one slot per 4 blocks of a row.  A slot comes round after kStages groups of at least one stage:
    // the last stage of the group that had it was filled again, so its MMAs are done, before the group that gets it was.
    static constexpr int kSlot = kNorms ? 20 : 12;
};
static_assert(PairShape<R8_COVERAGE, float, true>::kSmem + 8192 <= 232448 && PairShape<R8_PRODUCTS, __half, false>::kSmem + 512 <= 232448 &&
              PairShape<R8_PRODUCTS, float, false>::kSmem + 512 <= 232448, "shared memory");
// behind the accumulators and the slots: the scales of the norms' lane operand, 4 columns for each issuing warp.  Copies and MMAs of
// one thread keep their order, those of two do not: no warp writes columns that the other's MMAs read.
static_assert(2 * kPairCols + 6 * 20 + 2 * 4 <= 512 && 2 * kPairCols + 6 * 12 <= 512, "TMEM columns");

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
// rows of 16 bytes: one sequence (see tma_line)
__device__ __forceinline__ void pair_line(const uint32_t dst, const CUtensorMap* map, const int x, const uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.1d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2}], [%3];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(bar) : "memory");
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
__device__ __forceinline__ float max3(const float a, const float b, const float c) {
    float r;
    asm("max.ftz.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
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

// Digits and exponents of -|c|^2 / 2 for the pair kernel, `rows` (whole tiles) of them; and the n_h elements of h made ready: +inf, or
// (keep) what they hold, a NaN with its sign bit set, so that the minimum over bits leaves it (looking at h in the readers instead costs
// 500k x 256 by 10 000 centres 6 %, 1M x 16 by 576 18 %).
// |c|^2 = m 2^(E - 150) with 24 bits of m = sum_i d_i 16^i; the lane operand holds 2^-9, 2^-5, 2^-1, 2^3, 2^7, 2^7 with the
// scale 2^-15, so the codes are -d_0 .. -d_4, -16 d_5 and the scale 2^(E - 127): its byte is E.  Subnormal norms count as 0;
// NaN and infinity, and the columns past the last, get the NaN scale: never the largest.
__global__ void rows8_norm_digits_kernel(const float* __restrict__ norms, const int64_t n, const int64_t rows, unsigned char* digits,
                                         unsigned char* scales, float* h, const int64_t n_h, const int keep) {
    const int64_t step = (int64_t)gridDim.x * blockDim.x, at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (int64_t i = at; i < rows; i += step) {
        const unsigned bits = i < n ? __float_as_uint(__fadd_rn(__ldg(norms + i), 0.0f)) : 0x7fc00000u;      // (+ 0: no negative zero)
        const unsigned e = (bits >> 23) & 255u, m = e > 0u ? (bits & 0x7fffffu) | 0x800000u : 0u;
        uint4 q = make_uint4(0u, 0u, 0u, 0u);
        q.x = to_e4m3x2(-(float)(m & 15u), -(float)(m >> 4 & 15u)) | to_e4m3x2(-(float)(m >> 8 & 15u), -(float)(m >> 12 & 15u)) << 16;
        q.y = to_e4m3x2(-(float)(m >> 16 & 15u), -16.0f * (float)(m >> 20 & 15u));
        reinterpret_cast<uint4*>(digits)[i] = q;
        *reinterpret_cast<unsigned*>(scales + r8_scale_word(i, 0, 1)) = (bits & 0x80000000u) ? 255u : e;
    }
    if (!keep) {
        for (int64_t i = at; i < n_h; i += step) h[i] = __uint_as_float(0x7f800000u);
    } else {
        unsigned* bits = reinterpret_cast<unsigned*>(h);
        for (int64_t i = at; i < n_h; i += step)
            if (bits[i] > 0x7f800000u && bits[i] < 0x80000000u) bits[i] |= 0x80000000u;
    }
}

// Which tiles a pair works on, as segments [c0, c1) of column tiles of one lane tile.  All tiles stand in one sequence, lane
// tile by lane tile.  RUNS (coverage): the sequence is cut into equal runs, one per pair, so that a lane tile stays as long as
// it can.  Otherwise (products) tile by tile in turn: pairs that run at the same time share operands in L2 and write
// neighbouring parts of the result's rows (8192^3 to bfloat16: 408 us, in runs 511; 4096 x 100 000 x 128: 197, in runs 243).
struct PairSpan {
    int64_t lt, next;
    int c0, c1;
};
template <bool RUNS>
__device__ __forceinline__ PairSpan pair_span(const R8Job& job, const int64_t at, const int64_t last) {
    PairSpan s;
    s.lt = at / job.col_tiles;
    s.c0 = (int)(at - s.lt * job.col_tiles);
    s.c1 = !RUNS ? s.c0 + 1 : (last - at < job.col_tiles - s.c0 ? s.c0 + (int)(last - at) : job.col_tiles);
    s.next = RUNS ? at + (s.c1 - s.c0) : at + (gridDim.x >> 1);
    return s;
}

struct PairMaps { CUtensorMap lane, col, lane_sf, col_sf, norm, norm_sf, out; };

template <int WHAT, typename T, bool KEEP, bool NARROW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairWarps * 32, 1)
rows8_pair_kernel(const __grid_constant__ PairMaps maps, const R8Job job) {
    using S = PairShape<WHAT, T, KEEP>;
    constexpr int kStages = S::kStages;
    extern __shared__ unsigned char s_raw[];
    __shared__ uint64_t s_full[kStages], s_empty[kStages], s_acc_full[2], s_acc_empty[2], s_kept_full[2], s_kept_empty[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort_word;
    __shared__ __align__(1024) unsigned char s_power[S::kNorms ? 4096 + 512 : 16];      // the lane operand of the norms' step, and its scales
    const R8Bound s_abort{&s_abort_word, job.wait_ns};
    unsigned char* kept = reinterpret_cast<unsigned char*>(((uintptr_t)s_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* tiles = kept + S::kKept;

    const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;    // warp: known to be uniform
    const uint32_t rank = cluster_rank();
    const int64_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int64_t first = S::kNorms ? job.tiles * pair / pairs : pair, last = S::kNorms ? job.tiles * (pair + 1) / pairs : job.tiles;
    const int kblocks = (job.D + kR8Block - 1) / kR8Block;
    const uint32_t kept_slots = 2 * kblocks <= kPairKept ? 2 : 1;
    // Two warps issue, one for each accumulator, tile by tile in turn: the way of one warp through a tile (waits, scales, MMAs,
    // commits) is longer than the MMAs of a narrow tile take (D = 128: 860 clocks for 480).  Only where two tiles fit the
    // ring of stages.  A wait names the parity of a stage's fill, so it must not begin before the fill kStages earlier has
    // completed.  A warp that begins tile t + 1 has seen its accumulator free, so the readers are through tile t - 1 and every
    // fill up to that tile's last stage is complete; the stages of t + 1 end 2 kblocks later, and 2 kblocks <= kStages keeps
    // the fills kStages earlier among those.  Wider rows, whose MMAs take longer than their issue, have one issuing warp.
    const bool two = 2 * kblocks <= kStages;
    if (threadIdx.x == 0) {
        s_abort_word = 0;
        for (int i = 0; i < kStages; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_acc_full[i], 1);
            mbar_init(&s_acc_empty[i], 2 * kPairReaders);
            mbar_init(&s_kept_full[i], 1);
            mbar_init(&s_kept_empty[i], two ? 2 : 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (S::kNorms) {
        // 128 equal rows of 32 codes without a swizzle: 16 bytes of a row, 8 rows a group; the second 16 are 0
        for (int i = threadIdx.x; i < (4096 + 512) / 4; i += blockDim.x) {
            const unsigned codes = i < 512 && (i & 3) == 0 ? 0x50301001u : (i < 512 && (i & 3) == 1 ? 0x7070u : 0u);
            reinterpret_cast<unsigned*>(s_power)[i] = i >= 1024 ? 0x70707070u : codes;
        }
        if (threadIdx.x < kStages * 4) {
            unsigned char* first = tiles + kStages * S::kTile + (threadIdx.x >> 2) * S::kFirst;
            *reinterpret_cast<unsigned*>(first + kPairSf + kPairNormSf + kPairNormB + 4 * (threadIdx.x & 3)) = 0u;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    const int width = NARROW ? job.width : kR8Block;
    if (NARROW && width == 16) {
        if (KEEP)
            for (int i = 0; i < 2; ++i) zero_smem(kept + i * (kPairKept / 2) * kPairA + kR8Lanes * 64, kR8Lanes * 16);
        for (int i = 0; i < kStages; ++i) {
            if (!KEEP) zero_smem(tiles + i * S::kTile + kR8Lanes * 64, kR8Lanes * 16);
            zero_smem(tiles + (i + 1) * S::kTile - kPairB + kPairCols / 2 * 64, kPairCols / 2 * 16);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
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
        uint32_t n = 0, items = 0;
        bool ok = !job.stall;
        for (int64_t at = first; at < last && ok;) {
            const PairSpan sp = pair_span<S::kNorms>(job, at, last);
            at = sp.next;
            const int row = (int)(sp.lt * kPairLanes) + (int)rank * kR8Lanes;
            if (KEEP) {
                const uint32_t slot = items % kept_slots, round = items / kept_slots;
                if (round > 0 && !r8_wait_warp(&s_kept_empty[slot], (round - 1) & 1u, s_abort)) { ok = false; break; }
                const uint32_t bar = leader_addr(&s_kept_full[slot]), to = smem_u32(kept) + slot * (kPairKept / 2) * kPairA;
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(&s_kept_full[slot], 2 * kblocks * kR8Lanes * width);
                    if (NARROW && width == 16) pair_line(to, &maps.lane, 2 * row, bar);
                    else
                        for (int kb = 0; kb < kblocks; ++kb) pair_tile(to + kb * kPairA, &maps.lane, kb * kR8Block, row, bar);
                }
                __syncwarp();
                ++items;
            }
            for (int ct = sp.c0; ct < sp.c1 && ok; ++ct)
                for (int kb = 0; kb < kblocks; ++kb, ++n) {
                    if (n >= kStages && !r8_wait_warp(&s_empty[st], phase ^ 1u, s_abort)) { ok = false; break; }
                    const uint32_t a = smem_u32(tiles + st * S::kTile), sf = smem_u32(tiles + kStages * S::kTile + st * S::kFirst);
                    const uint32_t bar = leader_addr(&s_full[st]);
                    const bool scales = (kb & 3) == 0;
                    if (elect_one()) {
                        if (rank == 0) {
                            const int codes = ((KEEP ? 0 : kR8Lanes) + kPairCols / 2) * width;
                            const int norms = S::kNorms && kb == 0 ? kPairNormB + kPairNormSf : 0;
                            mbar_expect_tx(&s_full[st], 2 * (codes + (scales ? kPairSf : 0) + norms));
                        }
                        const int col = ct * kPairCols + (int)rank * (kPairCols / 2);
                        if (NARROW && width == 16) {
                            if (!KEEP) pair_line(a, &maps.lane, 2 * row, bar);
                            pair_line(a + S::kTile - kPairB, &maps.col, 2 * col, bar);
                        } else {
                            if (!KEEP) pair_tile(a, &maps.lane, kb * kR8Block, row, bar);
                            pair_tile(a + S::kTile - kPairB, &maps.col, kb * kR8Block, col, bar);
                        }
                        if (scales) {
                            pair_scales(sf, &maps.lane_sf, kb >> 2, row >> 7, bar);
                            pair_scales(sf + 512, &maps.col_sf, kb >> 2, ct * kPairCols >> 7, bar);
                        }
                        if (S::kNorms && kb == 0) {
                            pair_line(sf + kPairSf + kPairNormSf, &maps.norm, 2 * col, bar);
                            pair_scales(sf + kPairSf, &maps.norm_sf, 0, ct * kPairCols >> 7, bar);
                        }
                    }
                    __syncwarp();
                    if (++st == kStages) { st = 0; phase ^= 1u; }
                }
        }
        // the last releases of the stages reach both blocks: neither leaves before they have
        for (uint32_t k = n > kStages ? n - kStages : 0; k < n && ok; ++k) ok = r8_wait_warp(&s_empty[k % kStages], (k / kStages) & 1u, s_abort);
        // no copy may be in flight when the pair leaves (they all are complete unless a role gave up)
        if (!ok && rank == 0) {
            for (uint32_t k = n > kStages ? n - kStages : 0; k < n; ++k)
                for (int it = 0; it < (1 << 16) && !mbar_try(&s_full[k % kStages], (k / kStages) & 1u); ++it) {}
            for (uint32_t k = items > kept_slots ? items - kept_slots : 0; k < items; ++k)
                for (int it = 0; it < (1 << 16) && !mbar_try(&s_kept_full[k % kept_slots], (k / kept_slots) & 1u); ++it) {}
        }
    } else if (warp <= 2) {
        const uint32_t own = (uint32_t)warp - 1;
        if (rank == 0 && (two || own == 0)) {
            const uint32_t groups = (uint32_t)(kblocks + 3) >> 2;
            uint32_t n = 0, t = 0, items = 0;                       // stages, tiles and items so far, the other warp's among them
            bool ok = true, fresh = true;
            constexpr uint32_t kIdesc = ((uint32_t)(kPairCols >> 3) << 17) | (1u << 23) | ((uint32_t)(kPairLanes >> 4) << 24);
            const uint32_t base = smem_u32(tiles), power = smem_u32(s_power), sf_power = tmem + kSf + kStages * S::kSlot + 4 * own;
            for (int64_t at = first; at < last && ok;) {
                const PairSpan sp = pair_span<S::kNorms>(job, at, last);
                at = sp.next;
                const uint32_t kept_slot = items % kept_slots, kept_at = smem_u32(kept) + kept_slot * (kPairKept / 2) * kPairA;
                if (KEEP && !r8_wait_warp(&s_kept_full[kept_slot], items / kept_slots & 1u, s_abort)) { ok = false; break; }
                ++items;
                for (int ct = sp.c0; ct < sp.c1 && ok; ++ct, ++t) {
                    const uint32_t buf = t & 1u, round = t >> 1;
                    if (two && buf != own) {
                        n += (uint32_t)kblocks;
                        continue;
                    }
                    if (round > 0 && !r8_wait_warp(&s_acc_empty[buf], (round - 1) & 1u, s_abort)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t acc = tmem + buf * kPairCols;
                    // the tile's first column within its chunk of 128 scales: 32 rows a TMEM column
                    const uint32_t sub = (uint32_t)(ct * kPairCols & 127) >> 5;
                    uint32_t slot = t * groups % kStages, st = n % kStages, phase = n / kStages & 1u;
                    for (int kb = 0; kb < kblocks; ++kb, ++n) {
                        if (!r8_wait_warp(&s_full[st], phase, s_abort)) { ok = false; break; }
                        tc_fence_after();
                        if (kb > 0 && (kb & 3) == 0 && ++slot == kStages) slot = 0;
                        if (elect_one()) {
                            const uint32_t b = base + (st + 1) * S::kTile - kPairB, a = KEEP ? kept_at + kb * kPairA : b - kPairA;
                            const uint32_t sf = base + kStages * S::kTile + st * S::kFirst, norm = sf + kPairSf;
                            const uint32_t sfa = tmem + kSf + slot * S::kSlot, sfb = sfa + 4;
                            // (the lane operand's powers for the norms: by each warp before its own MMAs)
                            if (S::kNorms && fresh) pair_copy_scales(sf_power, umma_desc(power + 4096, 128, 0));
                            if ((kb & 3) == 0) {
                                pair_copy_scales(sfa, umma_desc(sf, 128, 0));
                                pair_copy_scales(sfb, umma_desc(sf + 512, 128, 0));
                                pair_copy_scales(sfb + 4, umma_desc(sf + 1024, 128, 0));
                            }
                            const uint32_t id = kIdesc | ((uint32_t)(kb & 3) << 4) | ((uint32_t)(kb & 3) << 29);
                            const int left = job.D - kb * kR8Block;
                            if (S::kNorms && kb == 0) {
                                // first: the sums that follow pass through 0 instead of growing to |a| |c|, and the accumulator
                                // loses less.  16 of the step's 32 codes count (the lane operand's others are 0): as the second 16 of
                                // a row the descriptor names the next row's digits, then the zero bytes
                                pair_copy_scales(sfb + 8, umma_desc(norm, 128, 0));
                                pair_copy_scales(sfb + 12, umma_desc(norm + 512, 128, 0));
                                pair_mma(acc, umma_desc(power, 128, 0) + (127ull << 16), umma_desc(norm + kPairNormSf, 128, 0), kIdesc, sf_power,
                                         sfb + 8 + sub, false);
                            }
                            // (NARROW kernels of their own: descriptors that the compiler knows but for the address issue 10 % faster)
                            if constexpr (!NARROW) {
                                const uint64_t da = umma_desc(a, 1024, 2), db = umma_desc(b, 1024, 2);
                                if (left > 96) {
#pragma unroll
                                    for (int k = 0; k < 4; ++k)
                                        pair_mma(acc, da + 2 * k, db + 2 * k, id, sfa, sfb + sub, S::kNorms || kb > 0 || k > 0);
                                } else {
                                    const int steps = (left + 31) >> 5;
                                    for (int k = 0; k < steps; ++k)
                                        pair_mma(acc, da + 2 * k, db + 2 * k, id, sfa, sfb + sub, S::kNorms || kb > 0 || k > 0);
                                }
                            } else {
                                const uint64_t da = tile_desc(a, width, kR8Lanes * 64), db = tile_desc(b, width, kPairCols / 2 * 64);
                                for (int k = 0; k < (left + 31) >> 5; ++k)
                                    pair_mma(acc, da + 2 * k, db + 2 * k, id, sfa, sfb + sub, S::kNorms || k > 0);
                            }
                            pair_commit(&s_empty[st]);
                            if (kb == kblocks - 1) pair_commit(&s_acc_full[buf]);
                        }
                        __syncwarp();
                        fresh = false;
                        if (++st == kStages) { st = 0; phase ^= 1u; }
                    }
                }
                // (only where the slot is filled again: nobody would wait for the last of these)
                if (KEEP && ok && (last - 1) / job.col_tiles - sp.lt >= kept_slots && elect_one()) pair_commit(&s_kept_empty[kept_slot]);
                __syncwarp();
            }
            // the tensor cores may still read the stages of a drained pair: wait for what was issued
            if (!ok)
                for (uint32_t k = n > kStages ? n - kStages : 0; k < n; ++k)
                    for (int it = 0; it < (1 << 16) && !mbar_try(&s_empty[k % kStages], (k / kStages) & 1u); ++it) {}
        }
    } else {
        const int quad = warp & 3, part = (warp - 3) >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16) + part * kPairPart;
        const float low = __uint_as_float(0xff800000u);
        uint32_t t = 0;
        bool ok = true;
        for (int64_t at = first; at < last && ok;) {
            const PairSpan sp = pair_span<S::kNorms>(job, at, last);
            at = sp.next;
            const int64_t row = sp.lt * kPairLanes + rank * kR8Lanes + quad * 32 + lane;
            float best[4] = {low, low, low, low};
            const float row_norm = WHAT == R8_COVERAGE && row < job.n_lane ? __ldg(job.lane_norms + row) : 0.0f;     // (ahead of the tiles)
            for (int ct = sp.c0; ct < sp.c1 && ok; ++ct, ++t) {
                const uint32_t buf = t & 1u;
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
                    if (job.bulk_out) {
                        // 48 columns x 32 lanes through shared memory, one bulk store for the warp (it leaves out what lies
                        // past the last lane or column)
                        T* mine = reinterpret_cast<T*>(tiles + kStages * (S::kTile + S::kFirst)) + (warp - 3) * (kPairPart * 32);
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < kPairPart; ++j) r8_narrow(mine[j * 32 + lane], __uint_as_float(v[j]));
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0 && row < job.n_lane && col < job.n_col) r8_store_tile(&maps.out, (int)row, (int)col, smem_u32(mine));
                    } else if (row < job.n_lane) {
                        T* out = reinterpret_cast<T*>(job.out) + row * job.lane_stride + col * job.col_stride;
#pragma unroll
                        for (int j = 0; j < kPairPart; ++j)
                            if (col + j < job.n_col) {
                                T o;
                                r8_narrow(o, __uint_as_float(v[j]));
                                r8_put(out + j * job.col_stride, o);
                            }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kPairPart; j += 2)
                        best[(j >> 1) & 3] = max3(best[(j >> 1) & 3], __uint_as_float(v[j]), __uint_as_float(v[j + 1]));
                }
            }
            if (WHAT == R8_COVERAGE && ok && row < job.n_lane) {
                // |a - c|^2 = |a|^2 - 2 (a.c - |c|^2 / 2)
                const float d = __fmaf_rn(-2.0f, fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3])), row_norm);
                // h holds +inf or what it had: a NaN leaves that, and so does whatever meets a NaN there, whose sign bit is set (see
                // rows8_norm_digits_kernel); max(d, 0) orders like its bits
                if (d == d)
                    atomicMin(reinterpret_cast<int*>(job.out) + row, __float_as_int(fmaxf(d, 0.0f)));
            }
        }
        if (WHAT == R8_PRODUCTS && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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
