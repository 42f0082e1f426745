// Rows in 8 bits: launchers and C entry points.
// Part of the single translation unit fps_kernels.cu (included there, last).
#ifndef CORESETS_B200_ROWS8_ENTRY_CUH
#define CORESETS_B200_ROWS8_ENTRY_CUH

namespace {

int validate_rows8(const cs_rows8* r) {
    if (!r || r->capacity < 0 || r->count < 0 || r->count > r->capacity || r->dim < 1 || (r->flags & ~CS_ROWS8_TEST_STALL)) return CS_E_ARG;
    if (r->capacity > 0 && (!r->codes || !r->scales || !r->norms)) return CS_E_ARG;
    if (r->capacity >= (int64_t)1 << 31 || r->dim > CS_ROWS8_MAX_DIM) return CS_E_RANGE;
    if (((uintptr_t)r->codes | (uintptr_t)r->scales | (uintptr_t)r->norms) & 15u) return CS_E_ALIGN;
    return CS_OK;
}

int r8_grid(const int64_t groups, const DevInfo& d) {
    const int64_t cap = (int64_t)d.sms * 8;                 // 2048 threads an SM
    return (int)(groups < 1 ? 1 : (groups < cap ? groups : cap));
}

// the widest load or store (16, 8, 4 or 2 bytes) that addresses, row stride and row length are whole multiples of
int r8_width(const void* p, const int64_t stride_bytes, const int64_t row_bytes) {
    const uintptr_t all = (uintptr_t)p | (uintptr_t)stride_bytes | (uintptr_t)row_bytes;
    return (all & 15u) == 0 ? 16 : ((all & 7u) == 0 ? 8 : ((all & 3u) == 0 ? 4 : 2));
}

template <typename T, int G, int U, bool ROWS>
int launch_rows8_write(const cs_rows8* r, const T* X, int64_t n, int64_t ld, int64_t start, cudaStream_t st, const DevInfo& d) {
    constexpr int kMid = sizeof(T) == 4 ? 8 : 4, kOne = (int)sizeof(T);
    const int width = r8_width(X, n > 1 ? ld * sizeof(T) : 0, (int64_t)r->dim * sizeof(T));
    const int64_t rows = (int64_t)(kThreads / G) * (ROWS && width == 16 ? U : 1);
    // many more blocks than fit at once: they even out what a block meets (2M x 256 float32: 428 us, 8 blocks an SM 448, one pass 467)
    const int64_t want = (n + rows - 1) / rows, most = (int64_t)d.sms * 64;
    const int grid = (int)(want < most ? want : most);
    if (width == 16) rows8_write_kernel<T, G, U, ROWS, 16><<<grid, kThreads, 0, st>>>(*r, X, n, ld, start);
    else if (width >= kMid) rows8_write_kernel<T, G, 1, ROWS, kMid><<<grid, kThreads, 0, st>>>(*r, X, n, ld, start);
    else rows8_write_kernel<T, G, 1, ROWS, kOne><<<grid, kThreads, 0, st>>>(*r, X, n, ld, start);
    return check_launch();
}
template <typename T>
int launch_rows8_write(const cs_rows8* r, const void* X, int64_t n, int64_t ld, int64_t start, cudaStream_t st, const DevInfo& d) {
    const T* x = static_cast<const T*>(X);
    if (((uintptr_t)X % sizeof(T)) != 0) return CS_E_ALIGN;
    // the lanes that 8 elements each of the row (its first block) take: padding codes up to the pitch are theirs too.
    // 64 bytes in flight a lane where loads are 16 bytes wide (4M x 128 float32: 442 us, one row at a time 555); narrow loads are
    // bound by their number and lose with fewer warps resident (2M x 50 float16: 116 us, four rows at a time 162)
    constexpr int U = sizeof(T) == 4 ? 2 : 4;
    if (r->dim <= 16) return launch_rows8_write<T, 2, U, true>(r, x, n, ld, start, st, d);
    if (r->dim <= 32) return launch_rows8_write<T, 4, U, true>(r, x, n, ld, start, st, d);
    if (r->dim <= 64) return launch_rows8_write<T, 8, U, true>(r, x, n, ld, start, st, d);
    if (r->dim <= 128) return launch_rows8_write<T, 16, U, true>(r, x, n, ld, start, st, d);
    return launch_rows8_write<T, 16, U, false>(r, x, n, ld, start, st, d);
}

template <typename T, int E, int G>
int launch_rows8_read(const cs_rows8* r, const int64_t* rows, int64_t m, T* out, int64_t ld, cudaStream_t st, const DevInfo& d) {
    constexpr int R = 4;                            // 2M x 256 to float32: 452 us; R = 2: 532, R = 8: 472
    const int64_t per_block = (int64_t)(kThreads / G) * R;
    rows8_read_kernel<T, E, G, R><<<r8_grid((m + per_block - 1) / per_block, d), kThreads, 0, st>>>(*r, rows, m, out, ld);
    return check_launch();
}
template <typename T, int E>
int launch_rows8_read(const cs_rows8* r, const int64_t* rows, int64_t m, T* out, int64_t ld, cudaStream_t st, const DevInfo& d) {
    const int chunks = r->dim / E;
    if (chunks <= 4) return launch_rows8_read<T, E, 4>(r, rows, m, out, ld, st, d);
    if (chunks <= 8) return launch_rows8_read<T, E, 8>(r, rows, m, out, ld, st, d);
    if (chunks <= 16) return launch_rows8_read<T, E, 16>(r, rows, m, out, ld, st, d);
    return launch_rows8_read<T, E, 32>(r, rows, m, out, ld, st, d);
}
template <typename T>
int launch_rows8_read(const cs_rows8* r, const int64_t* rows, int64_t m, void* out, int64_t ld, cudaStream_t st, const DevInfo& d) {
    T* o = static_cast<T*>(out);
    if (((uintptr_t)out % sizeof(T)) != 0) return CS_E_ALIGN;
    const int width = r8_width(out, m > 1 ? ld * sizeof(T) : 0, (int64_t)r->dim * sizeof(T));
    if (width == 16) return launch_rows8_read<T, 16 / (int)sizeof(T)>(r, rows, m, o, ld, st, d);
    if (width == 8) return launch_rows8_read<T, 8 / (int)sizeof(T)>(r, rows, m, o, ld, st, d);
    if (width == 4 && sizeof(T) == 2) return launch_rows8_read<T, 2>(r, rows, m, o, ld, st, d);
    return launch_rows8_read<T, 1>(r, rows, m, o, ld, st, d);
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

constexpr int64_t kR8LineRows = ((int64_t)1 << 30) - 1024;

// Bytes of a row in a tile: the narrowest swizzle that holds the row, 128 (a block) where none does.  A copy that is mostly
// past the end of its rows is slow, as is one that L2 widens past them (coverage of 1M x 16 by 576: 208 us with 128 bytes a row
// and 256 at a time from L2, 96 this way; by 16: 87 and 30).
// (16: as one sequence, whose places in units of 8 bytes have to fit 31 bits)
int r8_width_of(const int dim, const int64_t rows) { return dim <= 16 && rows <= kR8LineRows ? 16 : (dim <= 32 ? 32 : (dim <= 64 ? 64 : kR8Block)); }

// rows of `dim` bytes as tiles of `rows` x `width`; what lies behind the last row or the pitch reads as 0
int r8_map(CUtensorMap* map, void* base, const int dim, const int64_t count, const int width, const int rows) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return CS_E_DEVICE;
    const cuuint64_t dims[2] = {(cuuint64_t)r8_pitch(dim), (cuuint64_t)count};
    const cuuint64_t strides[1] = {(cuuint64_t)r8_pitch(dim)};
    const cuuint32_t box[2] = {(cuuint32_t)width, (cuuint32_t)rows}, step[2] = {1, 1};
    if (width == 16) {                                      // rows of 16 bytes, without a swizzle: one sequence, in units of 8 bytes
        const cuuint64_t all[1] = {(cuuint64_t)count * 2};
        const cuuint32_t part[1] = {(cuuint32_t)rows * 2};
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 1, base, all, strides, part, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
                   ? CS_OK
                   : CS_E_ARG;
    }
    const CUtensorMapSwizzle swizzle = width == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : (width == 64 ? CU_TENSOR_MAP_SWIZZLE_64B :
                                       CU_TENSOR_MAP_SWIZZLE_32B);
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? CS_OK
               : CS_E_ARG;
}

// the scale words of 128 rows as rows of 512 bytes, `chunks` consecutive tiles of 128 rows at once
int r8_scale_map(CUtensorMap* map, void* base, const int dim, const int64_t count, const int chunks) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return CS_E_DEVICE;
    const cuuint64_t words = (cuuint64_t)r8_words(dim);
    const cuuint64_t dims[3] = {128, words, (cuuint64_t)((count + 127) / 128)};
    const cuuint64_t strides[2] = {512, words * 512};
    const cuuint32_t box[3] = {128, 1, (cuuint32_t)chunks}, step[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? CS_OK
               : CS_E_ARG;
}

// Products leave by bulk stores of 32 lanes x `cols` where their rows follow the lanes and start and end on 16 bytes (a bulk
// store is cut off at whole 16 bytes, not at elements); bfloat16 16384 x 8192 x 256: 70 us, by the readers' own stores 150.
// Sets job.bulk_out.
template <typename T>
int r8_out_map(CUtensorMap* map, R8Job& job, const int cols) {
    job.bulk_out = job.lane_stride == 1 && ((uintptr_t)job.out & 15u) == 0 && (job.col_stride * sizeof(T)) % 16 == 0 &&
                   (job.n_lane * sizeof(T)) % 16 == 0 && job.col_stride >= job.n_lane;
    if (!job.bulk_out) return CS_OK;
    EncodeTiled encode = encode_tiled();
    if (!encode) return CS_E_DEVICE;
    const cuuint64_t dims[2] = {(cuuint64_t)job.n_lane, (cuuint64_t)job.n_col}, strides[1] = {(cuuint64_t)job.col_stride * sizeof(T)};
    const cuuint32_t box[2] = {32, (cuuint32_t)cols}, step[2] = {1, 1};
    return encode(map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, job.out, dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? CS_OK
               : CS_E_ARG;
}

// what the pair kernel's extra step needs per column, rounded up to whole tiles: 16 bytes of digits, then scale words
int64_t r8_norm_rows(const int64_t n_col) { return n_col <= 64 ? 0 : (n_col + kPairCols - 1) / kPairCols * kPairCols; }

template <int WHAT, typename T, bool KEEP, bool NARROW>
int launch_rows8_pair(const cs_rows8* lanes, const cs_rows8* cols, R8Job& job, void* work, cudaStream_t st, const DevInfo& d) {
    using S = PairShape<WHAT, T, KEEP>;
    PairMaps maps = {};
    int rc = r8_map(&maps.lane, lanes->codes, lanes->dim, lanes->count, job.width, kR8Lanes);
    if (!rc) rc = r8_map(&maps.col, cols->codes, cols->dim, cols->count, job.width, kPairCols / 2);
    if (!rc) rc = r8_scale_map(&maps.lane_sf, lanes->scales, lanes->dim, lanes->count, 1);
    if (!rc) rc = r8_scale_map(&maps.col_sf, cols->scales, cols->dim, cols->count, 2);
    if (rc) return rc;
    const int64_t pairs = d.sms / 2, lane_tiles = (job.n_lane + kPairLanes - 1) / kPairLanes;
    job.col_tiles = (int)((job.n_col + kPairCols - 1) / kPairCols);
    job.tiles = lane_tiles * job.col_tiles;
    if (S::kNorms) {
        const int64_t rows = r8_norm_rows(job.n_col);
        unsigned char* digits = static_cast<unsigned char*>(work);
        unsigned char* scales = digits + rows * 16;
        const int64_t most = rows > job.n_lane ? rows : job.n_lane;
        rows8_norm_digits_kernel<<<r8_grid((most + kThreads - 1) / kThreads, d), kThreads, 0, st>>>(
            job.col_norms, job.n_col, rows, digits, scales, static_cast<float*>(job.out), job.n_lane, job.keep);
        rc = check_launch();
        if (!rc) rc = r8_map(&maps.norm, digits, 16, rows, 16, kPairCols / 2);
        if (!rc) rc = r8_scale_map(&maps.norm_sf, scales, 1, rows, 2);
        if (rc) return rc;
    }
    if (!S::kNorms) {
        rc = r8_out_map<T>(&maps.out, job, kPairPart);
        if (rc) return rc;
    }
    static thread_local KernelTune tune;
    rc = tune_kernel(rows8_pair_kernel<WHAT, T, KEEP, NARROW>, tune, d.dev, S::kSmem, kPairWarps * 32, nullptr);
    if (rc) return rc;
    const int grid = 2 * (int)(job.tiles < pairs ? job.tiles : pairs);
    rows8_pair_kernel<WHAT, T, KEEP, NARROW><<<grid, kPairWarps * 32, S::kSmem, st>>>(maps, job);
    return check_launch();
}

template <int NT, int WHAT, typename T, bool NARROW>
int launch_rows8_mma_width(const cs_rows8* lanes, const cs_rows8* cols, R8Job& job, cudaStream_t st, const DevInfo& d) {
    using S = R8Shape<NT, WHAT, T>;
    CUtensorMap lane_map, col_map, out_map = {};
    int rc = r8_map(&lane_map, lanes->codes, lanes->dim, lanes->count, job.width, kR8Lanes);
    if (!rc) rc = r8_map(&col_map, cols->codes, cols->dim, cols->count, job.width, NT);
    if (!rc && WHAT == R8_PRODUCTS) rc = r8_out_map<T>(&out_map, job, NT);
    if (rc) return rc;
    static thread_local KernelTune tune;
    rc = tune_kernel(rows8_mma_kernel<NT, WHAT, T, NARROW>, tune, d.dev, S::kSmem, S::kThreads, nullptr);
    if (rc) return rc;
    job.items = (job.n_lane + kR8Lanes - 1) / kR8Lanes;
    const int grid = (int)(job.items < d.sms ? job.items : d.sms);
    rows8_mma_kernel<NT, WHAT, T, NARROW><<<grid, S::kThreads, S::kSmem, st>>>(lane_map, col_map, out_map, job);
    return check_launch();
}
template <int NT, int WHAT, typename T>
int launch_rows8_mma(const cs_rows8* lanes, const cs_rows8* cols, R8Job& job, cudaStream_t st, const DevInfo& d) {
    return job.width < kR8Block ? launch_rows8_mma_width<NT, WHAT, T, true>(lanes, cols, job, st, d)
                                : launch_rows8_mma_width<NT, WHAT, T, false>(lanes, cols, job, st, d);
}
// the narrowest tile that holds all columns; pairs of SMs where 64 do not (coverage of 1M x 128 by 8192 centres:
// 1.28 ms, with tiles of 128 x 128 on single SMs 3.11 ms)
template <int WHAT, typename T>
int launch_rows8_mma(const cs_rows8* lanes, const cs_rows8* cols, R8Job& job, void* work, cudaStream_t st, const DevInfo& d) {
    if (job.n_col <= 16) return launch_rows8_mma<16, WHAT, T>(lanes, cols, job, st, d);
    if (job.n_col <= 32) return launch_rows8_mma<32, WHAT, T>(lanes, cols, job, st, d);
    if (job.n_col <= 64) return launch_rows8_mma<64, WHAT, T>(lanes, cols, job, st, d);
    constexpr bool kMayKeep = WHAT == R8_COVERAGE;
    if (job.width < kR8Block) return launch_rows8_pair<WHAT, T, kMayKeep, true>(lanes, cols, job, work, st, d);
    if (kMayKeep && job.D <= kPairKept * kR8Block) return launch_rows8_pair<WHAT, T, kMayKeep, false>(lanes, cols, job, work, st, d);
    return launch_rows8_pair<WHAT, T, false, false>(lanes, cols, job, work, st, d);
}

R8Job r8_job(const cs_rows8* lanes, const cs_rows8* cols) {
    R8Job j = {};
    j.lane_scales = static_cast<const unsigned char*>(lanes->scales);
    j.col_scales = static_cast<const unsigned char*>(cols->scales);
    j.lane_norms = lanes->norms;
    j.col_norms = cols->norms;
    j.n_lane = lanes->count;
    j.n_col = cols->count;
    j.D = lanes->dim;
    j.words = r8_words(lanes->dim);
    j.width = r8_width_of(lanes->dim, lanes->count > cols->count ? lanes->count : cols->count);
    j.status = lanes->status;
    j.stall = (lanes->flags & CS_ROWS8_TEST_STALL) != 0;
    j.wait_ns = j.stall ? kR8TestWaitNs : kR8WaitNs;
    return j;
}

}  // namespace

extern "C" {

int cs_rows8_write(const cs_rows8* r, const void* X, int32_t dtype, int64_t n, int64_t ld, int64_t start, cs_stream stream) {
    int rc = validate_rows8(r);
    if (rc) return rc;
    if (n < 0 || start < 0 || start > r->capacity || n > r->capacity - start || (n > 0 && !X) || (n > 1 && ld < r->dim)) return CS_E_ARG;
    if (dtype < CS_DTYPE_F32 || dtype > CS_DTYPE_BF16) return CS_E_ARG;
    if (n == 0) return CS_OK;
    DevInfo d = device_info();
    if (!d.ok) return CS_E_DEVICE;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == CS_DTYPE_F32) return launch_rows8_write<float>(r, X, n, ld, start, st, d);
    if (dtype == CS_DTYPE_F16) return launch_rows8_write<__half>(r, X, n, ld, start, st, d);
    return launch_rows8_write<__nv_bfloat16>(r, X, n, ld, start, st, d);
}

int cs_rows8_read(const cs_rows8* r, const int64_t* rows, int64_t m, void* out, int32_t dtype, int64_t ld, cs_stream stream) {
    int rc = validate_rows8(r);
    if (rc) return rc;
    if (m < 0 || (m > 0 && !out) || (m > 1 && ld < r->dim) || (!rows && m > r->count)) return CS_E_ARG;
    if (dtype < CS_DTYPE_F32 || dtype > CS_DTYPE_BF16) return CS_E_ARG;
    if (m == 0) return CS_OK;
    DevInfo d = device_info();
    if (!d.ok) return CS_E_DEVICE;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == CS_DTYPE_F32) return launch_rows8_read<float>(r, rows, m, out, ld, st, d);
    if (dtype == CS_DTYPE_F16) return launch_rows8_read<__half>(r, rows, m, out, ld, st, d);
    return launch_rows8_read<__nv_bfloat16>(r, rows, m, out, ld, st, d);
}

int cs_rows8_take(const cs_rows8* src, const int64_t* rows, int64_t m, const cs_rows8* dst, int64_t start, cs_stream stream) {
    int rc = validate_rows8(src);
    if (rc) return rc;
    rc = validate_rows8(dst);
    if (rc) return rc;
    if (src->dim != dst->dim || m < 0 || (m > 0 && !rows) || start < 0 || start > dst->capacity || m > dst->capacity - start) return CS_E_ARG;
    if (m == 0) return CS_OK;
    if (src->codes == dst->codes || src->scales == dst->scales) return CS_E_ARG;
    DevInfo d = device_info();
    if (!d.ok) return CS_E_DEVICE;
    rows8_take_kernel<<<r8_grid((m + kWarps - 1) / kWarps, d), kThreads, 0, (cudaStream_t)stream>>>(*src, rows, m, *dst, start);
    return check_launch();
}

int cs_rows8_products(const cs_rows8* a, const cs_rows8* b, void* out, int32_t dtype, int64_t ld, cs_stream stream) {
    int rc = validate_rows8(a);
    if (rc) return rc;
    rc = validate_rows8(b);
    if (rc) return rc;
    if (a->dim != b->dim || dtype < CS_DTYPE_F32 || dtype > CS_DTYPE_BF16) return CS_E_ARG;
    if (a->count == 0 || b->count == 0) return CS_OK;
    if (!out || (a->count > 1 && ld < b->count)) return CS_E_ARG;
    if ((uintptr_t)out % (dtype == CS_DTYPE_F32 ? 4u : 2u)) return CS_E_ALIGN;
    DevInfo d = device_info();
    if (!d.ok) return CS_E_DEVICE;
    // lanes store consecutive elements of an output row when they are rows of b; with few rows of b most
    // of the 128 lanes would be empty
    const bool swap = b->count <= 64 && a->count > b->count;
    const cs_rows8* lanes = swap ? a : b;
    const cs_rows8* cols = swap ? b : a;
    R8Job job = r8_job(lanes, cols);
    job.status = a->status;
    job.out = out;
    job.lane_stride = swap ? ld : 1;
    job.col_stride = swap ? 1 : ld;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == CS_DTYPE_F32) return launch_rows8_mma<R8_PRODUCTS, float>(lanes, cols, job, nullptr, st, d);
    if (dtype == CS_DTYPE_F16) return launch_rows8_mma<R8_PRODUCTS, __half>(lanes, cols, job, nullptr, st, d);
    return launch_rows8_mma<R8_PRODUCTS, __nv_bfloat16>(lanes, cols, job, nullptr, st, d);
}

int64_t cs_rows8_coverage_bytes(int64_t n_centres) {
    if (n_centres < 0) return CS_E_ARG;
    const int64_t rows = r8_norm_rows(n_centres);
    return rows * 16 + (rows + 127) / 128 * 512;
}

int cs_rows8_coverage(const cs_rows8* a, const cs_rows8* centres, float* h, int32_t keep, void* work, cs_stream stream) {
    int rc = validate_rows8(a);
    if (rc) return rc;
    rc = validate_rows8(centres);
    if (rc) return rc;
    if (a->dim != centres->dim) return CS_E_ARG;
    if (centres->count > kR8LineRows) return CS_E_RANGE;
    if (a->count == 0) return CS_OK;
    if (!h) return CS_E_ARG;
    if ((uintptr_t)h & 3u) return CS_E_ALIGN;
    DevInfo d = device_info();
    if (!d.ok) return CS_E_DEVICE;
    cudaStream_t st = (cudaStream_t)stream;
    if (centres->count == 0) {
        if (keep) return CS_OK;
        rows8_fill_kernel<<<r8_grid((a->count + kThreads - 1) / kThreads, d), kThreads, 0, st>>>(h, a->count, __builtin_huge_valf());
        return check_launch();
    }
    if (r8_norm_rows(centres->count) > 0 && !work) return CS_E_ARG;
    if ((uintptr_t)work & 15u) return CS_E_ALIGN;
    R8Job job = r8_job(a, centres);
    job.out = h;
    job.keep = keep != 0;
    return launch_rows8_mma<R8_COVERAGE, float>(a, centres, job, work, st, d);
}

}  // extern "C"

#endif  // CORESETS_B200_ROWS8_ENTRY_CUH
