// C-ABI implementation of the training operators (include/hgemm_sm100_train.h):
// argument checks, tile choice, TMA descriptors and launches on the caller's
// stream. Descriptors are encoded per call and travel as kernel parameters.
#include "hgemm_sm100_train.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>

#include "train_kernels.cuh"

namespace {

using namespace hgemm;

__device__ int g_train_status_word;  // status word used when the caller passes none

constexpr int kMaxDevices = 64;
constexpr uint64_t kDefaultTimeoutNs = 2000ull * 1000ull * 1000ull;
constexpr int64_t kMaxSize = (int64_t{1} << 31) - 1024;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return cdiv(a, b) * b; }

struct DeviceInfo {
    int sms = 0;
    int* status_word = nullptr;
    int error = HGEMM_SM100_ERR_CUDA;
    std::once_flag once;
};
DeviceInfo g_devices[kMaxDevices];

int device_info(const DeviceInfo** out, int* id) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return HGEMM_SM100_ERR_CUDA;
    // Binds the device's context to this thread: a thread that has made no CUDA
    // call yet (autograd's) has none, and descriptor encoding needs it.
    if (cudaSetDevice(dev) != cudaSuccess) return HGEMM_SM100_ERR_CUDA;
    DeviceInfo& d = g_devices[dev];
    std::call_once(d.once, [&d, dev] {
        int major = 0, minor = 0;
        if (cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev) != cudaSuccess)
            return;
        if (major != 10 || minor != 0) {
            d.error = HGEMM_SM100_ERR_UNSUPPORTED_DEVICE;
            return;
        }
        if (cudaGetSymbolAddress(reinterpret_cast<void**>(&d.status_word), g_train_status_word) != cudaSuccess) return;
        d.error = HGEMM_SM100_OK;
    });
    *out = &d;
    *id = dev;
    return d.error;
}

// ------------------------------------------------------------ tensor maps --

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return static_cast<EncodeTiledFn>(nullptr);
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// Row-major matrix [rows x cols], pitch ld elements, in boxes of box_rows x
// box_cols; elements outside it read as zero and are not written.
int tensor_map(CUtensorMap* out, const void* base, int64_t cols, int64_t rows, int64_t ld, uint32_t box_cols,
               uint32_t box_rows, CUtensorMapDataType type, CUtensorMapSwizzle swizzle) {
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return HGEMM_SM100_ERR_TENSOR_MAP;
    const cuuint64_t esize = type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * esize};
    const cuuint32_t box[2] = {box_cols, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(out, type, 2, const_cast<void*>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? HGEMM_SM100_OK : HGEMM_SM100_ERR_TENSOR_MAP;
}

CUtensorMapDataType type16(int bf16) {
    return bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// ---------------------------------------------------------------- kernels --

using KernelFn = void (*)(TrainParams);
struct KernelEntry {
    KernelFn fn;
    std::atomic<uint64_t> ready{0};   // bit d: attributes set on device d
};
#define HG_TRAIN(PAIR, EPI) KernelEntry { &train_gemm_kernel<PAIR, EPI> }
KernelEntry g_kernels[2][6] = {
    {HG_TRAIN(false, kTrainStore), HG_TRAIN(false, kTrainGate), HG_TRAIN(false, kTrainGateGrad),
     HG_TRAIN(false, kTrainLse), HG_TRAIN(false, kTrainLogitGrad), HG_TRAIN(false, kTrainStoreC)},
    {HG_TRAIN(true, kTrainStore), HG_TRAIN(true, kTrainGate), HG_TRAIN(true, kTrainGateGrad),
     HG_TRAIN(true, kTrainLse), HG_TRAIN(true, kTrainLogitGrad), HG_TRAIN(true, kTrainStoreC)},
};

// Launch with programmatic stream serialisation (the kernels wait for the
// previous kernel before they touch global memory).
template <typename... P, typename... A>
int launch(void (*fn)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...) == cudaSuccess ? HGEMM_SM100_OK
                                                                                 : HGEMM_SM100_ERR_LAUNCH;
}

// ---------------------------------------------------------- one GEMM launch --

// An operand as it lies in memory. K-major: rows along M (or N), columns along
// K; MN-major: rows along K.
struct Operand {
    const void* ptr = nullptr;
    int64_t ld = 0;
    bool mn = false;
};

struct Tile {
    bool pair = false;
    int n = 0;
};

// One product as the host describes it. Two segments where k1 > 0; with `dual`
// b0 and b1 are the two column halves instead (n counts one half's columns).
struct Product {
    int64_t m = 0, n = 0, k0 = 0, k1 = 0;
    Operand a0, b0, a1, b1;
    bool dual = false;
    void* out = nullptr;       // 16-bit [m x ld_out]
    int64_t ld_out = 0;
    void* out1 = nullptr;      // further 16-bit outputs of the same shape
    void* out2 = nullptr;
    float alpha = 1.f, beta = 0.f;
    const float* alpha_ptr = nullptr;
    const float* alpha_rows = nullptr;
    const void* c = nullptr;
    int64_t ldc = 0;
    bool splittable = false;   // sums may be cut into parts
    bool symmetric = false;    // the product is symmetric (m == n)
    // Chosen with the tile: the last `parted` tiles in `splits` parts each, to
    // `parts` (FP32; added to what is there with add_parts); upper triangle only.
    int64_t parted = 0;
    int splits = 1;
    float* parts = nullptr;
    bool add_parts = false;
    bool triangle = false;
    // The sum's length that the raster goes by, where launches of different
    // lengths add to the same parts (a part's place is its tile's raster number).
    int64_t raster_k = 0;
    int64_t kblocks() const { return cdiv(k0, kBlockK) + cdiv(k1, kBlockK); }
};

// Cycles of one K block of 64 by tile, measured with every SM at work
// (2560 x 2560 x 9728 and 2560 x 9728 x 2560): a 256-wide pair tile comes near
// its MMAs' 512, narrow tiles meet the hand-off of a stage.
double block_cycles(bool pair, int tile_n) {
    static const double kSingle[4] = {310, 440, 560, 650}, kPairs[4] = {305, 335, 470, 595};
    return (pair ? kPairs : kSingle)[tile_n / 64 - 1];
}

int64_t tile_rows(bool pair) { return pair ? 256 : 128; }

int64_t tile_count(const Product& p, const Tile& t) {
    const int64_t rows = cdiv(p.m, tile_rows(t.pair)), cols = cdiv(p.n, p.dual ? t.n / 2 : t.n);
    return p.triangle ? rows * (rows + 1) / 2 : rows * cols;
}

double tile_time(int64_t kb, const Tile& t) { return static_cast<double>(kb) * block_cycles(t.pair, t.n) + 600.0; }

// Writing the parts of a product's last tiles, reading them, and one launch more.
double parts_time(const Product& p, const Tile& t) {
    return 6000.0 + 8.0 * p.splits * static_cast<double>(p.parted * tile_rows(t.pair) * t.n) / 3600.0;
}

// Parts of a product's sum for `want` parts: whole numbers of K blocks, none
// empty, at least `least` blocks in each.
int whole_parts(const Product& p, int64_t want, int64_t least) {
    const int64_t kb = p.kblocks(), most = std::max<int64_t>(1, kb / least);
    return static_cast<int>(cdiv(kb, cdiv(kb, std::min(want, most))));
}

// Operands' way from memory, 3600 bytes a cycle.
double memory_time(const Product& p) {
    return 2.0 * static_cast<double>(p.k0 + p.k1) * static_cast<double>(p.m + (p.dual ? 2 : 1) * p.n) / 3600.0;
}

double launch_time(const Tile& t) { return (t.pair ? 10000.0 : 8500.0) + 16.0 * t.n; }

// Time of one product with tile t: its full waves, and the last one, whose
// tiles may be cut into parts that fill it (or all tiles' parts, where there are
// fewer tiles than units). Sets the product's choices.
double plan_product(Product& p, const Tile& t, int sms, int forced_splits) {
    p.parted = 0;
    p.splits = 1;
    p.triangle = p.symmetric && t.n == tile_rows(t.pair);
    const int64_t units = t.pair ? sms / 2 : sms, tiles = tile_count(p, t), kb = p.kblocks();
    const int64_t rest = tiles % units;
    double best = static_cast<double>(cdiv(tiles, units)) * tile_time(kb, t);
    if (p.splittable && !p.triangle && (forced_splits != 0 || (rest != 0 && rest <= units / 2))) {
        Product q = p;
        q.parted = forced_splits != 0 && rest == 0 ? tiles : rest;
        for (int splits : {2, 3, 4, 5, 6, 8, 10, 12, 16}) {
            if (forced_splits != 0) splits = forced_splits;
            // Parts of four K blocks at least (of one where forced).
            q.splits = whole_parts(p, splits, forced_splits != 0 ? 1 : 4);
            if (q.splits < 2 && forced_splits == 0) break;
            const double time = static_cast<double>((tiles - q.parted) / units) * tile_time(kb, t) +
                                static_cast<double>(cdiv(q.parted * q.splits, units)) * tile_time(cdiv(kb, q.splits), t) +
                                parts_time(q, t);
            if (time < best || forced_splits != 0) {
                best = time;
                p.parted = q.parted;
                p.splits = q.splits;
            }
            if (forced_splits != 0 || q.parted * splits >= 2 * units) break;
        }
    }
    return std::max(best, memory_time(p)) + launch_time(t);
}

// Time of several products in one launch: units take the tiles one after the
// other, so the whole work over all units plus half a last tile that some wait
// for, and never less than the longest tile. A splittable product's tiles all
// come in `splits` parts (or whole, for 1).
double plan_group(Product* s, int count, const Tile& t, int sms, int splits) {
    double work = 0, longest = 0, last = 0, more = 0, memory = 0;
    for (int i = 0; i < count; ++i) {
        Product& p = s[i];
        p.triangle = p.symmetric && t.n == tile_rows(t.pair);
        p.splits = p.splittable ? splits : 1;
        p.parted = p.splits > 1 ? tile_count(p, t) : 0;
        const double one = tile_time(cdiv(p.kblocks(), p.splits), t);
        work += one * static_cast<double>(tile_count(p, t) * p.splits);
        longest = std::max(longest, one);
        last = one;
        memory += memory_time(p);
        if (p.splits > 1) more += parts_time(p, t);
    }
    return std::max({longest, work / (t.pair ? sms / 2 : sms) + 0.5 * last, memory}) + more + launch_time(t);
}

// The tile of a launch (all its products alike), and the products' parts.
Tile choose_tile(Product* s, int count, int sms, const HgemmSm100TrainCommon& forced) {
    const Product* split = nullptr;
    for (int i = 0; i < count; ++i)
        if (s[i].splittable) split = &s[i];
    Tile best;
    int best_splits = 1;
    double cost = -1;
    auto take = [&](const Tile& t, int splits, double c) {
        if (cost >= 0 && c >= cost) return;
        best = t;
        best_splits = splits;
        cost = c;
    };
    for (int pair = 1; pair >= 0; --pair) {
        for (int n = 256; n >= 64; n -= 64) {
            const Tile t{pair != 0, n};
            if (forced.tile != 0 && forced.tile != (n | (pair ? HGEMM_SM100_TRAIN_TILE_PAIR : 0))) continue;
            if (count == 1) {
                take(t, 1, plan_product(s[0], t, sms, forced.splits));
                continue;
            }
            double before = -1;
            for (int want : {1, 2, 3, 4, 6, 8, 12, 16}) {
                const int splits = split == nullptr      ? 1
                                   : forced.splits != 0 ? whole_parts(*split, forced.splits, 1)
                                                        : whole_parts(*split, want, 4);
                const double c = plan_group(s, count, t, sms, splits);
                take(t, splits, c);
                // More parts only as long as they help.
                if (split == nullptr || forced.splits != 0 || (before >= 0 && c >= before)) break;
                before = c;
            }
        }
    }
    if (count == 1) plan_product(s[0], best, sms, forced.splits);
    else plan_group(s, count, best, sms, best_splits);
    return best;
}

size_t parts_bytes(const Product& p, const Tile& t) {
    return static_cast<size_t>(p.parted) * p.splits * tile_rows(t.pair) * t.n * 4;
}

// Raster group height: the tallest of 8, 16, 32 tile rows whose one-wave
// footprint of A and B panels stays within 48 MB (the pair kernels' rule).
int group_height(const Product& p, bool pair, int sms) {
    const int64_t m = p.m, k = p.raster_k > 0 ? p.raster_k : p.k0 + p.k1;
    const int units = pair ? sms / 2 : sms;
    const int rows = pair ? 256 : 128;
    const double panel = 2.0 * rows * static_cast<double>(k);
    int g = 8;
    for (int h : {16, 32})
        if (h <= cdiv(m, rows) && (h + static_cast<double>(units) / h) * panel <= 48e6) g = h;
    return g;
}

int make_operand(CUtensorMap* map, const Operand& o, int64_t rows, int64_t k, uint32_t box_rows, int bf16) {
    return o.mn ? tensor_map(map, o.ptr, rows, k, o.ld, 64, 64, type16(bf16), CU_TENSOR_MAP_SWIZZLE_128B)
                : tensor_map(map, o.ptr, k, rows, o.ld, 64, box_rows, type16(bf16), CU_TENSOR_MAP_SWIZZLE_128B);
}

struct Context {
    const DeviceInfo* dev = nullptr;
    int id = 0;
    cudaStream_t stream = nullptr;
    HgemmSm100TrainCommon common{};
};

bool aligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool aligned16(const void* p) { return aligned(p, 16); }

int begin(Context* c, const HgemmSm100TrainCommon& common, void* stream) {
    if (!aligned(common.status, 4)) return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    if (common.dtype != HGEMM_SM100_TRAIN_F16 && common.dtype != HGEMM_SM100_TRAIN_BF16)
        return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    if (common.flags & ~HGEMM_SM100_FLAG_TEST_INJECT_TX) return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    if (common.splits < 0 || common.splits > 16) return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    if (common.tile != 0) {
        const int n = common.tile & 0xfff;
        if ((common.tile & ~(0xfff | HGEMM_SM100_TRAIN_TILE_PAIR)) || n < 64 || n > 256 || n % 64)
            return HGEMM_SM100_ERR_UNKNOWN_CONFIG;
    }
    c->stream = static_cast<cudaStream_t>(stream);
    c->common = common;
    return device_info(&c->dev, &c->id);
}

// Common fields of a launch.
void init_params(TrainParams& p, const Context& c) {
    std::memset(static_cast<void*>(&p), 0, sizeof(p));
    p.in_bf16 = p.out_bf16 = c.common.dtype == HGEMM_SM100_TRAIN_BF16;
    p.status = c.common.status != nullptr ? c.common.status : c.dev->status_word;
    p.timeout_ns = c.common.timeout_ns != 0 ? c.common.timeout_ns : kDefaultTimeoutNs;
    p.inject = (c.common.flags & HGEMM_SM100_FLAG_TEST_INJECT_TX) ? 1 : 0;
}

// Fills the problems of `p` from `count` products (the one with the longest
// sums first; one whose last tiles are parted makes two problems) and launches
// them as one grid.
int run_products(TrainParams& p, int epi, const Product* products, const Tile& tile, int count, const Context& c) {
    const bool pair = tile.pair;
    const int tile_n = tile.n;
    const int units = pair ? c.dev->sms / 2 : c.dev->sms;
    uint32_t a_bytes = 0, b_bytes = 0;
    int64_t total = 0, light = 0;
    int problems = 0;
    const int bf16 = p.in_bf16;
    for (int i = 0; i < 2 * count; ++i) {
        const Product& s = products[i / 2];
        const bool parted = i % 2 != 0;
        const int64_t all = tile_count(s, tile), tiles = parted ? s.parted : all - s.parted;
        if (tiles == 0) continue;
        if (problems == kTrainMaxProblems || all >= (int64_t{1} << 30)) return HGEMM_SM100_ERR_INVALID_ARGUMENT;
        TrainProblem& q = p.prob[problems++];
        const int cols = s.dual ? tile_n / 2 : tile_n;          // output columns of a tile
        const uint32_t b_box = static_cast<uint32_t>(s.dual || pair ? tile_n / 2 : tile_n);
        q.m = static_cast<int>(s.m);
        q.n = static_cast<int>(s.n);
        q.tile_n = tile_n;
        q.nkb0 = static_cast<int>(cdiv(s.k0, kBlockK));
        q.nkb = static_cast<int>(s.kblocks());
        q.a_mn = s.a0.mn;
        q.b_mn = s.b0.mn;
        q.tiles_m = static_cast<int>(cdiv(s.m, tile_rows(pair)));
        q.tiles_n = static_cast<int>(cdiv(s.n, cols));
        q.group_m = group_height(s, pair, c.dev->sms);
        q.symmetric = s.triangle;
        q.tile0 = static_cast<int>(parted ? all - s.parted : 0);
        q.tiles = static_cast<int>(tiles);
        q.splits = parted ? s.splits : 1;
        q.kb_split = static_cast<int>(cdiv(s.kblocks(), q.splits));
        q.parted = parted;
        q.out_kind = !parted ? kTrainOut16 : s.add_parts ? kTrainOutF32Add : kTrainOutF32;
        q.alpha = s.alpha;
        q.beta = parted ? 0.f : s.beta;   // the join adds it
        q.alpha_ptr = s.alpha_ptr;
        q.alpha_rows = s.alpha_rows;
        q.c = s.c;
        q.ldc = s.ldc;
        // Few rows (K-major): only those are loaded. What the MMA reads in place
        // of the others is some other part of the ring, and gives accumulator
        // rows that nothing stores.
        const uint32_t a_rows = s.a0.mn || pair ? 128u : static_cast<uint32_t>(std::min<int64_t>(128, round_up(s.m, 8)));
        q.a_tile_bytes = a_rows * 128u;
        int rc = make_operand(&q.a[0], s.a0, s.m, s.k0, a_rows, bf16);
        if (rc == HGEMM_SM100_OK) rc = make_operand(&q.b[0], s.b0, s.n, s.k0, b_box, bf16);
        if (rc == HGEMM_SM100_OK && s.dual) rc = make_operand(&q.b[1], s.b1, s.n, s.k0, b_box, bf16);
        if (rc == HGEMM_SM100_OK && s.k1 > 0) {
            rc = make_operand(&q.a[1], s.a1, s.m, s.k1, a_rows, bf16);
            if (rc == HGEMM_SM100_OK) rc = make_operand(&q.b[1], s.b1, s.n, s.k1, b_box, bf16);
        }
        if (rc == HGEMM_SM100_OK && parted)
            rc = tensor_map(&q.out[0], s.parts, tile_n, q.splits * tiles * tile_rows(pair), tile_n, 32, 32,
                            CU_TENSOR_MAP_DATA_TYPE_FLOAT32, CU_TENSOR_MAP_SWIZZLE_128B);
        void* const outs[3] = {s.out, s.out1, s.out2};
        for (int j = 0; j < 3 && rc == HGEMM_SM100_OK && !parted; ++j)
            if (outs[j] != nullptr)
                rc = tensor_map(&q.out[j], outs[j], s.n, s.m, s.ld_out, 32, 32, type16(p.out_bf16),
                                CU_TENSOR_MAP_SWIZZLE_64B);
        if (rc != HGEMM_SM100_OK) return rc;
        a_bytes = std::max(a_bytes, q.a_tile_bytes);
        b_bytes = std::max(b_bytes, static_cast<uint32_t>(round_up(pair ? tile_n / 2 : tile_n, 64) * 128));
        total += tiles * q.splits;
        if (problems > 1) light += tiles * q.splits;
    }
    if (total >= (int64_t{1} << 31)) return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    p.heavy_tiles = static_cast<int>(total - light);
    p.light_tiles = static_cast<int>(light);
    const int grid_units = static_cast<int>(std::min<int64_t>(total, units));
    if (light > 0 && p.heavy_tiles % grid_units != 0) {
        p.light_skip = static_cast<int>(static_cast<double>(p.prob[0].kb_split) / p.prob[1].kb_split + 0.5);
    }
    p.b_offset = a_bytes;
    p.block_stride = a_bytes + b_bytes;
    // Two K blocks to a stage where three stages fit: the hand-off of a stage
    // costs about 280 cycles whatever the tile's width.
    p.sub = kTrainRingBytes / (2 * p.block_stride) >= 3 ? 2 : 1;
    p.stages = static_cast<int>(std::min<uint32_t>(kTrainRingBytes / (p.sub * p.block_stride), kTrainMaxStages));

    KernelEntry& k = g_kernels[pair ? 1 : 0][epi];
    const uint64_t bit = 1ull << c.id;
    if (!(k.ready.load(std::memory_order_acquire) & bit)) {
        if (cudaFuncSetAttribute(reinterpret_cast<const void*>(k.fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(kTrainSmemBytes)) != cudaSuccess)
            return HGEMM_SM100_ERR_LAUNCH;
        k.ready.fetch_or(bit, std::memory_order_acq_rel);
    }
    return launch(k.fn, dim3(static_cast<unsigned>(grid_units * (pair ? 2 : 1))), dim3(kTrainThreads), kTrainSmemBytes,
                  pair ? 2 : 1, c.stream, p);
}

int run_product(TrainParams& p, int epi, Product& s, const Context& c) {
    return run_products(p, epi, &s, choose_tile(&s, 1, c.dev->sms, c.common), 1, c);
}

// The parted tiles of a product (if any), joined into its output.
int join_parts(const Product& s, const Tile& t, const Context& c, int in_bf16, int out_bf16) {
    if (s.parted == 0) return HGEMM_SM100_OK;
    JoinParams p{};
    p.parts = s.parts;
    p.splits = s.splits;
    p.tiles = static_cast<int>(s.parted);
    p.tile0 = static_cast<int>(tile_count(s, t) - s.parted);
    p.tile_m = static_cast<int>(tile_rows(t.pair));
    p.tile_n = t.n;
    p.tiles_m = static_cast<int>(cdiv(s.m, p.tile_m));
    p.tiles_n = static_cast<int>(cdiv(s.n, t.n));
    p.group_m = group_height(s, t.pair, c.dev->sms);
    p.m = static_cast<int>(s.m);
    p.n = static_cast<int>(s.n);
    p.alpha = s.alpha;
    p.beta = s.beta;
    p.alpha_ptr = s.alpha_ptr;
    p.alpha_rows = s.alpha_rows;
    p.c = s.c;
    p.ldc = s.ldc;
    p.out = s.out;
    p.ld_out = s.ld_out;
    p.in_bf16 = in_bf16;
    p.out_bf16 = out_bf16;
    const int64_t rows = std::min<int64_t>(p.tile_m, s.m), per_block = 256 / (t.n / 8);
    // Grid rows are limited to 65535; more tiles are taken by further launches.
    for (int first = 0; first < p.tiles; first += 65535) {
        JoinParams q = p;
        q.tile0 += first;
        q.parts += static_cast<int64_t>(first) * p.tile_m * p.tile_n;
        const int rc = launch(&join_parts_kernel, dim3(static_cast<unsigned>(cdiv(rows, per_block)),
                                                       static_cast<unsigned>(std::min(p.tiles - first, 65535))),
                              dim3(256), 0, 1, c.stream, q);
        if (rc != HGEMM_SM100_OK) return rc;
    }
    return HGEMM_SM100_OK;
}

// A single product, with its parts at `parts` (of parts_bytes).
int run_and_join(Product& s, const Tile& t, void* parts, const Context& c) {
    TrainParams p;
    init_params(p, c);
    s.parts = static_cast<float*>(parts);
    const int rc = run_products(p, kTrainStore, &s, t, 1, c);
    return rc != HGEMM_SM100_OK ? rc : join_parts(s, t, c, p.in_bf16, p.out_bf16);
}

bool size_ok(int64_t v) { return v > 0 && v <= kMaxSize; }
bool size8_ok(int64_t v) { return size_ok(v) && v % 8 == 0; }
// A matrix operand: present, aligned, its pitch a multiple of 8 and at least `cols`.
bool matrix_ok(const void* p, int64_t ld, int64_t cols) {
    return p != nullptr && aligned16(p) && ld >= cols && ld % 8 == 0;
}

}  // namespace

// ------------------------------------------------------------ feed-forward --

namespace {

bool ffn_sizes_ok(int64_t tokens, int64_t hidden, int64_t inter, int64_t out) {
    return size_ok(tokens) && size8_ok(hidden) && size8_ok(inter) && size8_ok(out);
}

// y = h Wd^T
Product ffn_down(const HgemmSm100FfnForward& a) {
    Product d;
    d.m = a.tokens;
    d.n = a.out;
    d.k0 = a.inter;
    d.a0 = {a.h, a.inter, false};
    d.b0 = {a.down, a.inter, false};
    d.out = a.y;
    d.ld_out = a.out;
    d.splittable = true;
    return d;
}

// The gradients that are wanted, the one with the longest sums first.
struct FfnGradPlan {
    Product s[4];
    int count = 0, dx = -1;
    Tile tile;
    size_t bytes() const { return dx >= 0 ? parts_bytes(s[dx], tile) : 0; }
};

FfnGradPlan plan_ffn_backward(const HgemmSm100FfnBackward& a, int sms) {
    FfnGradPlan g;
    if (a.dx != nullptr) {
        Product& q = g.s[g.count++];
        q.m = a.tokens;
        q.n = a.hidden;
        q.k0 = q.k1 = a.inter;
        q.a0 = {a.dgate_pre, a.inter, false};
        q.b0 = {a.gate, a.hidden, true};
        q.a1 = {a.dup_pre, a.inter, false};
        q.b1 = {a.up, a.hidden, true};
        q.out = a.dx;
        q.ld_out = a.hidden;
        q.splittable = true;
    }
    auto weight = [&](void* out, const void* left, int64_t ld_left, int64_t rows, const void* right, int64_t ld_right,
                      int64_t cols) {
        if (out == nullptr) return;
        Product& q = g.s[g.count++];
        q.m = rows;
        q.n = cols;
        q.k0 = a.tokens;
        q.a0 = {left, ld_left, true};
        q.b0 = {right, ld_right, true};
        q.out = out;
        q.ld_out = cols;
    };
    weight(a.dgate, a.dgate_pre, a.inter, a.inter, a.x, a.ldx, a.hidden);
    weight(a.dup, a.dup_pre, a.inter, a.inter, a.x, a.ldx, a.hidden);
    weight(a.ddown, a.dy, a.lddy, a.out, a.h, a.inter, a.inter);
    if (g.count == 0) return g;
    g.tile = choose_tile(g.s, g.count, sms, a.common);
    auto length = [](const Product& p) { return cdiv(p.kblocks(), p.splits); };
    for (int i = 1; i < g.count; ++i)
        for (int j = i; j > 0 && length(g.s[j]) > length(g.s[j - 1]); --j) std::swap(g.s[j], g.s[j - 1]);
    for (int i = 0; i < g.count; ++i)
        if (g.s[i].splittable) g.dx = i;
    return g;
}

}  // namespace

extern "C" size_t hgemm_sm100_ffn_forward_workspace(const HgemmSm100FfnForward* a) {
    Context c;
    if (a == nullptr || !ffn_sizes_ok(a->tokens, a->hidden, a->inter, a->out)) return 0;
    if (begin(&c, a->common, nullptr) != HGEMM_SM100_OK) return 0;
    Product d = ffn_down(*a);
    const Tile t = choose_tile(&d, 1, c.dev->sms, c.common);
    return parts_bytes(d, t);
}

extern "C" int hgemm_sm100_ffn_forward(const HgemmSm100FfnForward* a, void* stream) {
    if (a == nullptr || !ffn_sizes_ok(a->tokens, a->hidden, a->inter, a->out)) return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    if (!matrix_ok(a->x, a->ldx, a->hidden) || !matrix_ok(a->gate, 8, 8) || !matrix_ok(a->up, 8, 8) ||
        !matrix_ok(a->down, 8, 8) || !matrix_ok(a->y, 8, 8) || !matrix_ok(a->h, 8, 8))
        return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    if ((a->silu == nullptr) != (a->slope == nullptr) || !aligned16(a->silu) || !aligned16(a->slope))
        return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    Context c;
    int rc = begin(&c, a->common, stream);
    if (rc != HGEMM_SM100_OK) return rc;
    Product d = ffn_down(*a);
    const Tile down_tile = choose_tile(&d, 1, c.dev->sms, c.common);
    const size_t need = parts_bytes(d, down_tile);
    if (need > 0 && (a->workspace == nullptr || !aligned16(a->workspace) || a->workspace_bytes < need))
        return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    TrainParams p;

    Product g;
    g.m = a->tokens;
    g.n = a->inter;
    g.k0 = a->hidden;
    g.a0 = {a->x, a->ldx, false};
    g.b0 = {a->gate, a->hidden, false};
    g.b1 = {a->up, a->hidden, false};
    g.dual = true;
    g.out = a->h;
    g.out1 = a->silu;
    g.out2 = a->slope;
    g.ld_out = a->inter;
    init_params(p, c);
    p.keep = a->silu != nullptr;
    if ((rc = run_product(p, kTrainGate, g, c)) != HGEMM_SM100_OK) return rc;

    return run_and_join(d, down_tile, a->workspace, c);
}

extern "C" size_t hgemm_sm100_ffn_backward_workspace(const HgemmSm100FfnBackward* a) {
    Context c;
    if (a == nullptr || !ffn_sizes_ok(a->tokens, a->hidden, a->inter, a->out)) return 0;
    if (begin(&c, a->common, nullptr) != HGEMM_SM100_OK) return 0;
    return plan_ffn_backward(*a, c.dev->sms).bytes();
}

extern "C" int hgemm_sm100_ffn_backward(const HgemmSm100FfnBackward* a, void* stream) {
    if (a == nullptr || !ffn_sizes_ok(a->tokens, a->hidden, a->inter, a->out)) return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    if (!matrix_ok(a->dy, a->lddy, a->out) || !matrix_ok(a->x, a->ldx, a->hidden) || !matrix_ok(a->gate, 8, 8) ||
        !matrix_ok(a->up, 8, 8) || !matrix_ok(a->down, 8, 8) || !matrix_ok(a->silu, 8, 8) ||
        !matrix_ok(a->slope, 8, 8) || !matrix_ok(a->h, 8, 8) || !matrix_ok(a->dgate_pre, 8, 8) ||
        !matrix_ok(a->dup_pre, 8, 8) || !aligned16(a->dx) || !aligned16(a->dgate) || !aligned16(a->dup) ||
        !aligned16(a->ddown))
        return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    Context c;
    int rc = begin(&c, a->common, stream);
    if (rc != HGEMM_SM100_OK) return rc;
    FfnGradPlan g = plan_ffn_backward(*a, c.dev->sms);
    const size_t need = g.bytes();
    if (need > 0 && (a->workspace == nullptr || !aligned16(a->workspace) || a->workspace_bytes < need))
        return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    if (g.count == 0) return HGEMM_SM100_OK;
    TrainParams p;

    // dh = dy Wd; its epilogue turns it into dg and du.
    if (a->dx != nullptr || a->dgate != nullptr || a->dup != nullptr) {
        Product h;
        h.m = a->tokens;
        h.n = a->inter;
        h.k0 = a->out;
        h.a0 = {a->dy, a->lddy, false};
        h.b0 = {a->down, a->inter, true};
        h.out = a->dgate_pre;
        h.out1 = a->dup_pre;
        h.ld_out = a->inter;
        init_params(p, c);
        p.silu = a->silu;
        p.slope = a->slope;
        p.ld_kept = a->inter;
        if ((rc = run_product(p, kTrainGateGrad, h, c)) != HGEMM_SM100_OK) return rc;
    }
    if (g.dx >= 0) g.s[g.dx].parts = static_cast<float*>(a->workspace);
    init_params(p, c);
    if ((rc = run_products(p, kTrainStore, g.s, g.tile, g.count, c)) != HGEMM_SM100_OK || g.dx < 0) return rc;
    return join_parts(g.s[g.dx], g.tile, c, p.in_bf16, p.out_bf16);
}

// ------------------------------------------------------------ cross entropy --

namespace {

struct LossForwardPlan {
    Product z;
    Tile tile;
    int64_t parts = 0;
    size_t partial_bytes = 0, row_bytes = 0;
    size_t bytes() const { return partial_bytes + 2 * row_bytes; }
};

LossForwardPlan plan_loss_forward(const HgemmSm100LossForward& a, int sms) {
    LossForwardPlan q;
    q.z.m = a.tokens;
    q.z.n = a.vocab;
    q.z.k0 = a.hidden;
    q.z.a0 = {a.x, a.ldx, false};
    q.z.b0 = {a.weight, a.hidden, false};
    q.tile = choose_tile(&q.z, 1, sms, a.common);
    q.parts = 2 * cdiv(a.vocab, q.tile.n);   // two column groups a tile
    q.partial_bytes = static_cast<size_t>(round_up(q.parts * a.tokens * 8, 256));
    q.row_bytes = static_cast<size_t>(round_up(a.tokens * 4, 256));
    return q;
}

// How the logits' gradient is scaled (logit_grad_setup_kernel).
int loss_scale(const HgemmSm100LossBackward& a) {
    if (a.reduction != HGEMM_SM100_LOSS_NONE) return kScaleOne;
    if (a.common.dtype == HGEMM_SM100_TRAIN_BF16) return kScaleBf16;
    return a.dx != nullptr ? kScaleRows : kScaleCommon;
}

// Rows of their own scale serve dx; dW needs dz in the common one as well.
int64_t loss_planes(const HgemmSm100LossBackward& a) {
    return loss_scale(a) == kScaleRows && a.dweight != nullptr ? 2 : 1;
}

// Vocabulary entries of a piece: as many as keep its dz (tokens x piece, 16
// bits, once or twice) within 96 MB, so that it stays in L2 between the product
// that writes it and the two that read it, in whole 256-column tiles, at least
// 2048.
int64_t loss_piece(const HgemmSm100LossBackward& a) {
    if (a.piece > 0) return std::min<int64_t>(round_up(a.piece, 8), round_up(a.vocab, 8));
    int64_t n = (int64_t{96} << 20) / (2 * loss_planes(a) * a.tokens) / 256 * 256;
    n = std::max<int64_t>(n, 2048);
    if (n >= a.vocab) return round_up(a.vocab, 8);
    return round_up(cdiv(a.vocab, cdiv(a.vocab, n)), 256);   // equal pieces
}

// dx and dW of one piece (nv vocabulary entries), as long sums first.
struct LossPiece {
    Product s[2];
    int count = 0, dx = -1;
    Tile tile;
};

LossPiece plan_piece(const HgemmSm100LossBackward& a, int64_t nv, int64_t piece, int sms) {
    LossPiece g;
    if (a.dx != nullptr) {
        Product& d = g.s[g.count++];
        d.m = a.tokens;
        d.n = d.ld_out = a.hidden;
        d.k0 = nv;
        d.raster_k = piece;   // a short last piece adds to the tiles of the others
        d.a0 = {nullptr, piece, false};
        d.b0 = {nullptr, a.hidden, true};
        d.splittable = true;
    }
    if (a.dweight != nullptr) {
        Product& d = g.s[g.count++];
        d.m = nv;
        d.n = d.ld_out = a.hidden;
        d.k0 = a.tokens;
        d.a0 = {nullptr, piece, true};
        d.b0 = {a.x, a.ldx, true};
    }
    g.tile = choose_tile(g.s, g.count, sms, a.common);
    return g;
}

struct LossBackwardPlan {
    int64_t piece = 0, pieces = 0;
    bool sums = false;     // dx goes through FP32 sums: several pieces, or parts of one
    int splits = 1;        // of dx, in every piece alike
    Tile tile;
    int64_t planes = 1;    // of dz
    size_t dz_bytes = 0, sum_bytes = 0, row_bytes = 0;   // of one plane, of dx, of one number per row
    size_t x_bytes = 0;    // x without the ignored rows
    size_t bytes() const { return planes * dz_bytes + sum_bytes + 3 * row_bytes + 256 + x_bytes; }
};

LossBackwardPlan plan_loss_backward(const HgemmSm100LossBackward& a, int sms) {
    LossBackwardPlan q;
    q.piece = loss_piece(a);
    q.pieces = cdiv(a.vocab, q.piece);
    q.planes = loss_planes(a);
    q.dz_bytes = static_cast<size_t>(round_up(a.tokens * q.piece * 2, 256));
    q.row_bytes = static_cast<size_t>(round_up(a.tokens * 4, 256));
    if (a.dweight != nullptr) q.x_bytes = static_cast<size_t>(a.tokens * a.hidden * 2);
    if (a.dx == nullptr && a.dweight == nullptr) return q;
    const int64_t last = a.vocab - (q.pieces - 1) * q.piece;
    const LossPiece g = plan_piece(a, std::min(q.piece, a.vocab), q.piece, sms);
    q.tile = g.tile;
    if (a.dx != nullptr) {
        // In whole pieces and the last one alike, each part has K blocks.
        auto parts_ok = [](int64_t n, int64_t splits) {
            const int64_t kb = cdiv(n, kBlockK);
            return (splits - 1) * cdiv(kb, splits) < kb;
        };
        q.splits = g.s[0].splits;
        while (!parts_ok(std::min(q.piece, a.vocab), q.splits) || !parts_ok(last, q.splits)) --q.splits;
        // Several pieces add up in FP32 tiles, in as many parts.
        Product d = g.s[0];
        d.splits = q.splits;
        if (q.pieces > 1 || q.splits > 1) d.parted = tile_count(d, q.tile);
        else d.parted = 0;
        q.sums = d.parted > 0;
        q.sum_bytes = static_cast<size_t>(round_up(static_cast<int64_t>(parts_bytes(d, q.tile)), 256));
    }
    return q;
}

template <typename Args>
bool loss_args_ok(const Args& a) {
    return size_ok(a.tokens) && size8_ok(a.hidden) && size_ok(a.vocab) && matrix_ok(a.x, a.ldx, a.hidden) &&
           matrix_ok(a.weight, 8, 8) && a.target != nullptr && aligned(a.target, 8) && a.lse != nullptr &&
           aligned(a.lse, 4) &&
           a.reduction >= HGEMM_SM100_LOSS_NONE && a.reduction <= HGEMM_SM100_LOSS_SUM;
}

}  // namespace

extern "C" size_t hgemm_sm100_loss_forward_workspace(const HgemmSm100LossForward* a) {
    Context c;
    if (a == nullptr || !size_ok(a->tokens) || !size_ok(a->vocab) || !size8_ok(a->hidden)) return 0;
    if (begin(&c, a->common, nullptr) != HGEMM_SM100_OK) return 0;
    return plan_loss_forward(*a, c.dev->sms).bytes();
}

extern "C" int hgemm_sm100_loss_forward(const HgemmSm100LossForward* a, void* stream) {
    if (a == nullptr || !loss_args_ok(*a) || a->loss == nullptr || !aligned(a->loss, 4) ||
        a->workspace == nullptr || !aligned16(a->workspace))
        return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    Context c;
    int rc = begin(&c, a->common, stream);
    if (rc != HGEMM_SM100_OK) return rc;
    const LossForwardPlan q = plan_loss_forward(*a, c.dev->sms);
    if (a->workspace_bytes < q.bytes()) return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    float2* partial = reinterpret_cast<float2*>(ws);
    float* target_logit = reinterpret_cast<float*>(ws + q.partial_bytes);
    float* rows = reinterpret_cast<float*>(ws + q.partial_bytes + q.row_bytes);
    float* loss = a->reduction == HGEMM_SM100_LOSS_NONE ? a->loss : rows;
    const int m = static_cast<int>(a->tokens);
    const long long* target = reinterpret_cast<const long long*>(a->target);

    TrainParams p;
    init_params(p, c);
    p.target = target;
    p.partial = partial;
    p.target_logit = target_logit;
    if ((rc = run_products(p, kTrainLse, &q.z, q.tile, 1, c)) != HGEMM_SM100_OK) return rc;
    rc = launch(&lse_join_kernel<8>, dim3(static_cast<unsigned>(cdiv(m, 8))), dim3(8, 128), 0, 1, c.stream, partial,
                static_cast<int>(q.parts), m, target_logit, target, static_cast<long long>(a->vocab),
                static_cast<long long>(a->ignore_index), a->lse, loss);
    if (rc != HGEMM_SM100_OK || a->reduction == HGEMM_SM100_LOSS_NONE) return rc;
    return launch(&loss_reduce_kernel, dim3(1), dim3(1024), 0, 1, c.stream, rows, target, m,
                  static_cast<long long>(a->ignore_index), a->reduction == HGEMM_SM100_LOSS_MEAN ? 1 : 0, a->loss);
}

extern "C" size_t hgemm_sm100_loss_backward_workspace(const HgemmSm100LossBackward* a) {
    Context c;
    if (a == nullptr || !size_ok(a->tokens) || !size_ok(a->vocab) || !size8_ok(a->hidden) || a->piece < 0) return 0;
    if (begin(&c, a->common, nullptr) != HGEMM_SM100_OK) return 0;
    return plan_loss_backward(*a, c.dev->sms).bytes();
}

extern "C" int hgemm_sm100_loss_backward(const HgemmSm100LossBackward* a, void* stream) {
    if (a == nullptr || !loss_args_ok(*a) || a->dloss == nullptr || !aligned(a->dloss, 4) || a->workspace == nullptr ||
        !aligned16(a->workspace) || !aligned16(a->dx) || !aligned16(a->dweight) || a->piece < 0)
        return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    Context c;
    int rc = begin(&c, a->common, stream);
    if (rc != HGEMM_SM100_OK) return rc;
    const LossBackwardPlan q = plan_loss_backward(*a, c.dev->sms);
    if (a->workspace_bytes < q.bytes()) return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    if (a->dx == nullptr && a->dweight == nullptr) return HGEMM_SM100_OK;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    uint8_t* dz = ws;                                          // as dx takes it
    uint8_t* dz_common = ws + (q.planes - 1) * q.dz_bytes;     // as dW does
    float* sums = reinterpret_cast<float*>(ws + q.planes * q.dz_bytes);
    uint8_t* rows = ws + q.planes * q.dz_bytes + q.sum_bytes;
    float* row_scale = reinterpret_cast<float*>(rows);
    float* row_alpha = reinterpret_cast<float*>(rows + q.row_bytes);
    float* row_ratio = reinterpret_cast<float*>(rows + 2 * q.row_bytes);
    float* alpha = reinterpret_cast<float*>(rows + 3 * q.row_bytes);
    void* x_kept = rows + 3 * q.row_bytes + 256;
    const int scale = loss_scale(*a);
    // What takes the factors out of dx.
    auto scale_dx = [&](Product& d) {
        if (scale == kScaleRows) d.alpha_rows = row_alpha;
        else d.alpha_ptr = alpha;
    };
    const long long* target = reinterpret_cast<const long long*>(a->target);

    // Copying blocks: four 16-byte pieces a thread, two waves of blocks at most.
    const int64_t copying = a->dweight == nullptr
                                ? 0
                                : std::min<int64_t>(cdiv(a->tokens * (a->hidden / 8), 4096), 4 * c.dev->sms);
    rc = launch(&logit_grad_setup_kernel, dim3(static_cast<unsigned>(1 + copying)), dim3(1024), 0, 1, c.stream, a->dloss,
                scale, a->reduction == HGEMM_SM100_LOSS_MEAN ? 1 : 0, target, static_cast<int>(a->tokens),
                static_cast<long long>(a->vocab), static_cast<long long>(a->ignore_index), row_scale, row_alpha,
                row_ratio, alpha, a->x, static_cast<long long>(a->ldx), static_cast<int>(a->hidden), x_kept);
    if (rc != HGEMM_SM100_OK) return rc;

    TrainParams p;
    for (int64_t i = 0; i < q.pieces; ++i) {
        const int64_t v0 = i * q.piece, nv = std::min(q.piece, a->vocab - v0);
        const uint8_t* w = static_cast<const uint8_t*>(a->weight) + v0 * a->hidden * 2;
        Product z;
        z.m = a->tokens;
        z.n = nv;
        z.k0 = a->hidden;
        z.a0 = {a->x, a->ldx, false};
        z.b0 = {w, a->hidden, false};
        z.out = dz;
        z.out1 = q.planes == 2 ? dz_common : nullptr;
        z.ld_out = q.piece;
        init_params(p, c);
        p.target = target;
        p.col_base = v0;
        p.lse = a->lse;
        p.row_scale = row_scale;
        p.row_ratio = q.planes == 2 ? row_ratio : nullptr;
        if ((rc = run_product(p, kTrainLogitGrad, z, c)) != HGEMM_SM100_OK) return rc;

        LossPiece g = plan_piece(*a, nv, q.piece, c.dev->sms);
        int n = 0;
        if (a->dx != nullptr) {
            Product& d = g.s[n++];
            d.a0.ptr = dz;
            d.b0.ptr = w;
            d.splits = q.splits;
            d.parted = q.sums ? tile_count(d, q.tile) : 0;
            d.parts = sums;
            d.add_parts = i > 0;
            d.out = a->dx;
            scale_dx(d);
        }
        if (a->dweight != nullptr) {
            Product& d = g.s[n++];
            d.a0.ptr = dz_common;
            d.b0 = {x_kept, a->hidden, true};
            d.out = static_cast<uint8_t*>(a->dweight) + v0 * a->hidden * 2;
            d.alpha_ptr = alpha;
        }
        if (n == 2 && g.s[1].kblocks() > cdiv(g.s[0].kblocks(), g.s[0].splits)) std::swap(g.s[0], g.s[1]);
        init_params(p, c);
        if ((rc = run_products(p, kTrainStore, g.s, q.tile, n, c)) != HGEMM_SM100_OK) return rc;
    }
    if (!q.sums) return HGEMM_SM100_OK;
    Product d = plan_piece(*a, std::min(q.piece, a->vocab), q.piece, c.dev->sms).s[0];
    d.splits = q.splits;
    d.parted = tile_count(d, q.tile);
    d.parts = sums;
    d.out = a->dx;
    scale_dx(d);
    return join_parts(d, q.tile, c, p.in_bf16, p.out_bf16);
}

// ------------------------------------------------------ orthogonalised update --

namespace {

constexpr int kOrthSums = 592;   // partial sums of squares per matrix, at most

struct OrthPlan {
    bool tall = false;
    int64_t side = 0, ld = 0, ld_side = 0, x_stride = 0, side_stride = 0;
    size_t sum_bytes = 0, x_bytes = 0, side_bytes = 0, parts_bytes = 0;
    size_t bytes() const { return sum_bytes + 2 * x_bytes + 2 * side_bytes + parts_bytes; }
};

// The three products of a step, with their sizes only.
Product orth_product(const HgemmSm100Orthogonalize& a, int which) {
    const int64_t side = std::min(a.rows, a.cols);
    Product s;
    s.m = which < 2 ? side : a.rows;
    s.n = which < 2 ? side : a.cols;
    s.k0 = which == 0 ? std::max(a.rows, a.cols) : side;
    s.symmetric = which < 2;
    s.splittable = which != 1 && a.batch == 1;
    return s;
}

OrthPlan plan_orth(const HgemmSm100Orthogonalize& a, int sms) {
    OrthPlan q;
    q.tall = a.rows > a.cols;
    q.side = std::min(a.rows, a.cols);
    q.ld = round_up(a.cols, 64);
    q.ld_side = round_up(q.side, 64);
    q.x_stride = a.rows * q.ld;
    q.side_stride = q.side * q.ld_side;
    q.sum_bytes = static_cast<size_t>(round_up(a.batch * kOrthSums * 8, 256));
    q.x_bytes = static_cast<size_t>(round_up(a.batch * q.x_stride * 2, 256));
    q.side_bytes = static_cast<size_t>(round_up(a.batch * q.side_stride * 2, 256));
    for (int which : {0, 2}) {
        Product s = orth_product(a, which);
        if (!s.splittable) continue;
        const Tile t = choose_tile(&s, 1, sms, a.common);
        q.parts_bytes = std::max(q.parts_bytes, static_cast<size_t>(round_up(static_cast<int64_t>(parts_bytes(s, t)), 256)));
    }
    return q;
}

// The one-launch form for a shorter side of at most 128 rows: CTAs of a cluster
// (each 128 rows x `slice` columns), 0 where it does not fit. The fewest with
// slices of at most 256 columns: a step's exchange between CTAs costs about 3 us
// and 256 columns of a step 3.8 (128 x 640: 50, 48, 43, 44 and 46 us with 1 to
// 16 CTAs; 128 x 256: 27 and 35 with 1 and 2).
int orth_cluster_ctas(const HgemmSm100Orthogonalize& a) {
    const int64_t side = std::min(a.rows, a.cols), length = std::max(a.rows, a.cols);
    if (a.common.tile != 0 || a.steps < 1 || side > 128) return 0;
    for (int n : {1, 2, 4, 8, 16}) {
        const int64_t slice = round_up(cdiv(length, n), 64);
        if (a.common.splits != 0 ? a.common.splits == n && slice <= kOrthMaxSlice
                                 : slice <= 256 || (n == 16 && slice <= kOrthMaxSlice))
            return n;
    }
    return 0;
}

using OrthFn = void (*)(OrthClusterParams);
struct OrthEntry {
    OrthFn fn;
    std::atomic<uint64_t> ready{0};
};
OrthEntry g_orth[5] = {{&orth_cluster_kernel<1>},
                       {&orth_cluster_kernel<2>},
                       {&orth_cluster_kernel<4>},
                       {&orth_cluster_kernel<8>},
                       {&orth_cluster_kernel<16>}};

int run_orth_cluster(const HgemmSm100Orthogonalize& a, int ctas, const Context& c) {
    OrthEntry& k = g_orth[ctas == 1 ? 0 : ctas == 2 ? 1 : ctas == 4 ? 2 : ctas == 8 ? 3 : 4];
    const uint64_t bit = 1ull << c.id;
    if (!(k.ready.load(std::memory_order_acquire) & bit)) {
        const void* fn = reinterpret_cast<const void*>(k.fn);
        if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kOrthMaxSmem)) !=
                cudaSuccess ||
            cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
            return HGEMM_SM100_ERR_LAUNCH;
        k.ready.fetch_or(bit, std::memory_order_acq_rel);
    }
    OrthClusterParams p{};
    p.g = a.g;
    p.out = a.out;
    p.batch_stride = a.batch_stride;
    p.ld = a.ldg;
    p.side = static_cast<int>(std::min(a.rows, a.cols));
    p.length = static_cast<int>(std::max(a.rows, a.cols));
    p.tall = a.rows > a.cols;
    p.slice = static_cast<int>(round_up(cdiv(p.length, ctas), 64));
    p.bf16 = a.common.dtype == HGEMM_SM100_TRAIN_BF16;
    // Rows of g and out in 16-byte pieces. A slice begins at a multiple of 64.
    p.vec_in = aligned16(a.g) && a.cols % 8 == 0 && a.ldg % 8 == 0 && a.batch_stride % 8 == 0;
    p.vec_out = aligned16(a.out) && a.cols % 8 == 0;
    p.steps = a.steps;
    p.a = a.a;
    p.b = a.b;
    p.c = a.c;
    p.eps = a.eps;
    p.status = a.common.status != nullptr ? a.common.status : c.dev->status_word;
    p.timeout_ns = a.common.timeout_ns != 0 ? a.common.timeout_ns : kDefaultTimeoutNs;
    // One CTA to an SM: two of different clusters would wait for the one's TMEM
    // while their clusters wait for them.
    const size_t smem = std::max<size_t>(
        static_cast<size_t>(p.slice / 64) * kOrthBlockBytes + 2 * kOrthSquareBytes + 1024 + 512, 120 * 1024);
    return launch(k.fn, dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(a.batch)),
                  dim3(kOrthThreads), smem, ctas, c.stream, p);
}

bool orth_sizes_ok(const HgemmSm100Orthogonalize& a) {
    return a.batch > 0 && a.batch <= 65535 && size_ok(a.rows) && size_ok(a.cols) && a.steps >= 0;
}

}  // namespace

extern "C" size_t hgemm_sm100_orthogonalize_workspace(const HgemmSm100Orthogonalize* a) {
    Context c;
    if (a == nullptr || !orth_sizes_ok(*a) || orth_cluster_ctas(*a) > 0) return 0;
    if (begin(&c, a->common, nullptr) != HGEMM_SM100_OK) return 0;
    return plan_orth(*a, c.dev->sms).bytes();
}

extern "C" int hgemm_sm100_orthogonalize(const HgemmSm100Orthogonalize* a, void* stream) {
    if (a == nullptr || !orth_sizes_ok(*a) || a->g == nullptr || a->out == nullptr || !aligned(a->g, 2) ||
        !aligned(a->out, 2) || a->ldg < a->cols || a->batch_stride < 0 || !(a->eps >= 0))
        return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    const int ctas = orth_cluster_ctas(*a);
    if (ctas == 0 && (a->workspace == nullptr || !aligned(a->workspace, 256)))
        return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    Context c;
    int rc = begin(&c, a->common, stream);
    if (rc != HGEMM_SM100_OK) return rc;
    if (ctas > 0) return run_orth_cluster(*a, ctas, c);
    const OrthPlan q = plan_orth(*a, c.dev->sms);
    if (a->workspace_bytes < q.bytes()) return HGEMM_SM100_ERR_INVALID_ARGUMENT;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    double* sums = reinterpret_cast<double*>(ws);
    uint16_t* x = reinterpret_cast<uint16_t*>(ws + q.sum_bytes);
    uint16_t* y = reinterpret_cast<uint16_t*>(ws + q.sum_bytes + q.x_bytes);
    uint16_t* gram = reinterpret_cast<uint16_t*>(ws + q.sum_bytes + 2 * q.x_bytes);
    uint16_t* poly = reinterpret_cast<uint16_t*>(ws + q.sum_bytes + 2 * q.x_bytes + q.side_bytes);
    float* parts = reinterpret_cast<float*>(ws + q.sum_bytes + 2 * q.x_bytes + 2 * q.side_bytes);
    const int bf16 = a->common.dtype == HGEMM_SM100_TRAIN_BF16 ? 1 : 0;
    const int rows = static_cast<int>(a->rows), cols = static_cast<int>(a->cols);
    // A block per 2048 elements, several waves of blocks at most.
    const unsigned blocks =
        static_cast<unsigned>(std::min<int64_t>(cdiv(a->rows * cdiv(a->cols, 8), 256), kOrthSums));
    const unsigned batch = static_cast<unsigned>(a->batch);

    const bool vec = aligned16(a->g) && a->cols % 8 == 0 && a->ldg % 8 == 0 && a->batch_stride % 8 == 0;
    rc = launch(vec ? &orth_square_kernel<true> : &orth_square_kernel<false>, dim3(blocks, batch), dim3(256), 0, 1,
                c.stream, a->g, static_cast<long long>(a->batch_stride), rows, cols, static_cast<long long>(a->ldg),
                bf16, sums);
    if (rc != HGEMM_SM100_OK) return rc;
    rc = launch(vec ? &orth_scale_kernel<true> : &orth_scale_kernel<false>, dim3(2 * blocks, batch), dim3(256), 0, 1,
                c.stream, a->g, static_cast<long long>(a->batch_stride), rows, cols, static_cast<long long>(a->ldg),
                bf16, sums, static_cast<int>(blocks), a->eps, reinterpret_cast<__half*>(x),
                static_cast<long long>(q.ld), static_cast<long long>(q.x_stride));
    if (rc != HGEMM_SM100_OK) return rc;

    // The last step writes the result itself where TMA can store it.
    const bool direct = aligned16(a->out) && a->cols % 8 == 0;
    const float inv = 1.f / kOrthScale;
    TrainParams p;
    // Product `which` of every matrix, up to four to a launch; make() adds the operands.
    auto each = [&](int which, auto&& make, int out_bf16) -> int {
        for (int64_t first = 0; first < a->batch; first += kTrainMaxProblems) {
            Product s[kTrainMaxProblems];
            const int n = static_cast<int>(std::min<int64_t>(kTrainMaxProblems, a->batch - first));
            for (int i = 0; i < n; ++i) {
                s[i] = orth_product(*a, which);
                make(s[i], first + i);
                s[i].parts = parts;
            }
            const Tile t = choose_tile(s, n, c.dev->sms, c.common);
            init_params(p, c);
            p.in_bf16 = 0;
            p.out_bf16 = out_bf16;
            int r = run_products(p, s[0].c != nullptr ? kTrainStoreC : kTrainStore, s, t, n, c);
            if (r == HGEMM_SM100_OK && n == 1) r = join_parts(s[0], t, c, 0, out_bf16);
            if (r != HGEMM_SM100_OK) return r;
        }
        return HGEMM_SM100_OK;
    };
    for (int step = 0; step < a->steps; ++step) {
        const bool last = step + 1 == a->steps;
        // gram = X X^T or X^T X
        rc = each(0, [&](Product& s, int64_t i) {
            const uint16_t* xi = x + i * q.x_stride;
            s.a0 = {xi, q.ld, q.tall};
            s.b0 = {xi, q.ld, q.tall};
            s.out = gram + i * q.side_stride;
            s.ld_out = q.ld_side;
            s.alpha = inv * inv;
        }, 0);
        if (rc != HGEMM_SM100_OK) return rc;
        // poly = b gram + c gram gram (symmetric)
        rc = each(1, [&](Product& s, int64_t i) {
            const uint16_t* gi = gram + i * q.side_stride;
            s.a0 = {gi, q.ld_side, false};
            s.b0 = {gi, q.ld_side, false};
            s.out = poly + i * q.side_stride;
            s.ld_out = q.ld_side;
            s.alpha = a->c;
            s.beta = a->b;
            s.c = gi;
            s.ldc = q.ld_side;
        }, 0);
        if (rc != HGEMM_SM100_OK) return rc;
        // X <- a X + poly X, or a X + X poly
        rc = each(2, [&](Product& s, int64_t i) {
            const uint16_t* xi = x + i * q.x_stride;
            const uint16_t* pi = poly + i * q.side_stride;
            if (q.tall) {
                s.a0 = {xi, q.ld, false};
                s.b0 = {pi, q.ld_side, false};
            } else {
                s.a0 = {pi, q.ld_side, false};
                s.b0 = {xi, q.ld, true};
            }
            s.c = xi;
            s.ldc = q.ld;
            s.alpha = last ? inv : 1.f;
            s.beta = last ? a->a * inv : a->a;
            if (last && direct) {
                s.out = static_cast<uint16_t*>(a->out) + i * a->rows * a->cols;
                s.ld_out = a->cols;
            } else {
                s.out = y + i * q.x_stride;
                s.ld_out = q.ld;
            }
        }, last ? bf16 : 0);
        if (rc != HGEMM_SM100_OK) return rc;
        std::swap(x, y);
    }
    if (direct && a->steps > 0) return HGEMM_SM100_OK;
    const bool none = a->steps == 0;
    return launch(&orth_copy_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(a->rows, 65535)), batch), dim3(256),
                  0, 1, c.stream, x, static_cast<long long>(q.ld), static_cast<long long>(q.x_stride),
                  none ? 0 : bf16, none ? inv : 1.f, a->out, rows, cols, bf16);
}

extern "C" int hgemm_sm100_train_read_status(int32_t* value, int clear) {
    const DeviceInfo* dev = nullptr;
    int id = 0;
    const int rc = device_info(&dev, &id);
    if (rc != HGEMM_SM100_OK) return rc;
    if (value != nullptr && cudaMemcpy(value, dev->status_word, sizeof(int32_t), cudaMemcpyDeviceToHost) != cudaSuccess)
        return HGEMM_SM100_ERR_CUDA;
    if (clear && cudaMemset(dev->status_word, 0, sizeof(int32_t)) != cudaSuccess) return HGEMM_SM100_ERR_CUDA;
    return HGEMM_SM100_OK;
}
