// sm_100a kernels of the training operators (gated feed-forward block and its
// gradient, cross entropy from hidden states and its gradient, orthogonalised
// updates). All of their matrix products run on one tcgen05 kernel template,
//
//   train_gemm_kernel<kPair, kEpi>:  acc[m, n] = sum_k A(m, k) B(k, n)
//
// for FP16 or BF16 operands and FP32 accumulators in TMEM. It differs from the
// inference kernels of hgemm_kernels.cuh in what a training step needs:
//
//  * either operand lies either way in memory (rows along K, "K-major", or
//    rows along M / N, "MN-major"), chosen per problem at run time: only the
//    TMA boxes and the matrix descriptors differ, so x W^T, dy W and dy^T x
//    all read the tensors where they are, without a transposed copy;
//  * the sum over K may run over two operand pairs (dx = dg Wg + du Wu), and
//    the columns of B may come from two tensors (gate and up), so no weight is
//    packed: a training step changes the weights every time;
//  * the last tiles' sums over K may be cut into parts, whose FP32 sums
//    join_parts_kernel adds in a fixed order: all tiles where there are fewer
//    than SMs (few rows, long sums), else those of a nearly empty last wave;
//  * of a symmetric product only the tiles on and above the diagonal are
//    computed, and stored both ways;
//  * one launch takes up to four problems and walks their tiles as one list
//    (dx, dWgate, dWup and dWdown fill the last wave together);
//  * the epilogue finishes the operator (SwiGLU, its gradient, softmax
//    statistics, the logits' gradient, a x X + acc) on the FP32 accumulators.
//
// kPair: tiles of 256 x tile_n per CTA pair (cta_group::2); otherwise 128 x
// tile_n per CTA. tile_n is a run-time multiple of 64 up to 256, which the host
// picks by what the waves of tiles are estimated to take.
// Roles per CTA: warps 0-7 epilogue (one TMEM lane = one output row per
// thread; warps w and w + 4 share a row quarter and take every second group of
// 32 columns), warp 8 TMA producer, warp 9 MMA issuer; two accumulators, so a
// tile's epilogue runs under the next tile's MMAs; eight warps, because the last
// tile's epilogue is exposed and the gradient of the gate is a long one (dh at
// 4096 x 9728 x 2560: 278 us with four, 192 with eight, 168 since its side inputs
// come in coalesced patches). Every wait is bounded
// as in the inference kernels (status word, drained copies, freed TMEM).
//
// What bounds it (2048 tokens, hidden 2560, under ncu): the tensor pipe where
// the epilogue stores nothing (softmax statistics: 91 % active, 1.66 PFLOP/s);
// 82-85 % where it stores 16 bits (logit gradients, the weights' gradients);
// 75 % with three outputs (gate); 50 % where it reads two matrices and writes
// two (gradient of the gate). DRAM is at 11-24 % and L2 at 43-54 % throughout.
// Long back-to-back runs are held by the power limit instead (sampled: 1.24 to
// 1.55 GHz of 1.965, the power cap active all the time; 1.2-1.35 PFLOP/s). A K block of a 256 x 256 pair tile takes about
// 590 cycles of which the MMAs are 512.
#pragma once

#include <cuda_bf16.h>

#include "hgemm_kernels.cuh"

namespace hgemm {

constexpr int kTrainMaxProblems = 4;   // of one launch
constexpr uint32_t kTrainRingBytes = 196608;               // stages of both operands
constexpr uint32_t kTrainBoxBytes = 2048;                  // 32 rows x 32 16-bit columns
constexpr int kTrainEpiWarps = 8;
constexpr int kTrainThreads = (kTrainEpiWarps + 2) * 32;
constexpr uint32_t kTrainEpiBytes = kTrainEpiWarps * 2u * kTrainBoxBytes;  // 2 boxes a warp
constexpr int kTrainMaxStages = 12;
constexpr uint32_t kTrainDataBytes = kTrainRingBytes + kTrainEpiBytes;
constexpr uint32_t kTrainSmemBytes = kTrainDataBytes + 256 + 1024;
constexpr uint32_t kTrainAccCols = 256;                    // TMEM columns per accumulator
static_assert(2 * kTrainMaxStages + 5 <= 30, "barrier area");
static_assert(kTrainSmemBytes <= 232448, "shared memory");

enum : int {
    kTrainStore = 0,      // out = alpha acc (16 bits), or FP32 acc stored / added
    kTrainGate = 1,       // acc = (gate | up): out = silu(gate) up; silu(gate) and up silu'(gate) kept
    kTrainGateGrad = 2,   // acc = dh: out = dh (up silu'(gate)), out[1] = dh silu(gate), from what was kept
    kTrainLse = 3,        // per row: max and sum of exp over the tile's columns
    kTrainLogitGrad = 4,  // out = (exp(acc - lse) - [column == target]) row factor; out[1] with another factor
    kTrainStoreC = 5,     // kTrainStore with out = alpha acc + beta C
};
// How kTrainStore and kTrainStoreC write: 16-bit boxes, FP32 boxes, FP32 boxes added to memory.
enum : int { kTrainOut16 = 0, kTrainOutF32 = 1, kTrainOutF32Add = 2 };

struct alignas(64) TrainProblem {
    CUtensorMap a[2];      // A of the first and second K segment
    CUtensorMap b[2];      // B of the two segments, or (dual) the two column halves
    CUtensorMap out[3];
    int m, n;              // output rows and columns (dual: columns of one half)
    int tile_n;            // accumulator columns of a tile (dual: both halves)
    int nkb0, nkb;         // K blocks of the first segment, of both
    int a_mn, b_mn;
    int tiles_m, tiles_n, group_m;
    int symmetric;         // tiles are those of the upper triangle, row by row
    int tile0, tiles;      // this problem's tiles of all: tile0 .. tile0 + tiles - 1
    int splits, kb_split;  // parts of the sum over K, K blocks of each (the last: the rest)
    int parted;            // out[0] holds FP32 tiles, [part][tile][rows of a tile][tile_n]
    uint32_t a_tile_bytes; // what the loads of A bring per K block
    int out_kind;
    float alpha, beta;
    const float* alpha_ptr;    // multiplies alpha (device memory; may be null)
    const float* alpha_rows;   // kTrainStore: multiplies alpha, per row (may be null)
    const void* c;             // FP16 [m x ldc] for beta != 0
    long long ldc;
};

struct alignas(64) TrainParams {
    TrainProblem prob[kTrainMaxProblems];
    int heavy_tiles, light_tiles;  // tiles of problem 0 / of the others
    int light_skip;                // waves the units with one heavy tile more sit out
    int stages, sub;               // ring stages, K blocks of 64 in each
    uint32_t block_stride;         // bytes of one K block's tiles in a stage
    uint32_t b_offset;             // where B starts among them
    int in_bf16, out_bf16;
    int* status;
    unsigned long long timeout_ns;
    int inject;                    // test only: arm the first stage with 16 bytes more
    // kTrainGateGrad: what the forward pass kept, 16-bit [m x ld_kept].
    const void* silu;              // silu(gate)
    const void* slope;             // up silu'(gate)
    long long ld_kept;
    int keep;                      // kTrainGate: store these too (out[1], out[2])
    // kTrainLse / kTrainLogitGrad, per row.
    const long long* target;
    long long col_base;            // vocabulary index of column 0
    float2* partial;               // kTrainLse: [2 tiles_n][m] (max, sum of exp(x - max))
    float* target_logit;           // kTrainLse: written by the tile holding the target
    const float* lse;
    const float* row_scale;
    const float* row_ratio;        // kTrainLogitGrad: out[1] = row_ratio out[0] too (may be null)
};

// ------------------------------------------------------------- small parts ---

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, int bf16) {
    return bf16 ? pack2<true>(lo, hi) : pack2<false>(lo, hi);
}
__device__ __forceinline__ float2 unpack2(uint32_t w, int bf16) {
    if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float to_f32(const void* base, long long i, int bf16) {
    return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i])
                : __half2float(static_cast<const __half*>(base)[i]);
}

// 2^x (about 2 ulp; -inf -> 0, NaN -> NaN).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// sigmoid(x), both approximations good to 2^-22; x -> -inf gives 0 (1 / (1 + inf)).
__device__ __forceinline__ float sigmoid_f(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + exp2_fast(-x * kLog2e)));
    return y;
}

// 32 16-bit values of one row, loaded ahead of their use. 16-byte-aligned
// vectors, read only where they hold elements of the row (rows are padded to a
// multiple of 8 elements); the others are zero.
struct Row32 {
    uint4 w[4];
    __device__ __forceinline__ void load(const void* base, long long off, int avail) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + off);
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = 8 * q < avail ? src[q] : make_uint4(0u, 0u, 0u, 0u);
    }
    template <bool kBf16>
    __device__ __forceinline__ float2 pair(int i) const {   // elements 2i, 2i + 1
        const uint4& v = w[i >> 2];
        return unpack2((i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w, kBf16);
    }
};

// A 32 x 32 patch of a 16-bit matrix in a warp's registers, loaded ahead of its
// use: lane l holds 16 bytes (columns 8 (l % 4) ..) of rows l / 4, l / 4 + 8, ...
// Four lanes share a row's 64 bytes, so a load touches 8 lines, not 32.
struct Patch32 {
    uint4 w[4];
    // Element (row0, col0) is the patch's first; rows and columns from `rows`,
    // `cols` on (counted from there) are zero. cols is a multiple of 8.
    __device__ __forceinline__ void load(const void* base, long long ld, int row0, int col0, int rows, int cols, uint32_t lane) {
        const int r = static_cast<int>(lane >> 2), c = static_cast<int>(lane & 3u) * 8;
        const uint16_t* src = static_cast<const uint16_t*>(base) + (row0 + r) * ld + col0 + c;
#pragma unroll
        for (int i = 0; i < 4; ++i, src += 8 * ld)
            w[i] = r + 8 * i < rows && c < cols ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
    }
    // Into a box (64-byte rows, swizzled as BoxWriter's).
    __device__ __forceinline__ void put(uint8_t* box, uint32_t lane) const {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t r = (lane >> 2) + 8u * i;
            *reinterpret_cast<uint4*>(box + r * 64u + (((lane & 3u) ^ ((r >> 1) & 3u)) << 4)) = w[i];
        }
    }
};

// Adds a 2-D box in shared memory to FP32 global memory (elements outside the
// map are not written).
__device__ __forceinline__ void tma_reduce_add_2d(const CUtensorMap* map, const void* src, int32_t x, int32_t y) {
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(src)), "r"(x), "r"(y)
                 : "memory");
}

// One epilogue warp's output boxes: 32 rows (lane = row) x 32 columns through
// shared memory to a TMA store, 16-bit boxes in two 2 KB buffers in turn
// (64-byte swizzle), FP32 boxes in one of 4 KB (128-byte swizzle). Before a
// buffer is rewritten, the store that used it last must have read it. Every
// value is rounded here, once.
struct BoxWriter {
    uint8_t* bufs;
    uint32_t next;
    uint32_t lane;
    bool whole;    // the last group of stores reads both buffers

    // The next buffer, once the store that used it last has read it.
    __device__ __forceinline__ uint8_t* take() {
        if (lane == 0) {
            if (whole) bulk_wait_group_read<0>();
            else bulk_wait_group_read<1>();
        }
        whole = false;
        __syncwarp();
        return bufs + (next++ & 1u) * kTrainBoxBytes;
    }
    template <bool kBf16>
    __device__ __forceinline__ void fill(uint8_t* box, const float (&v)[32]) const {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            uint4 q;
            q.x = pack2<kBf16>(v[8 * j + 0], v[8 * j + 1]);
            q.y = pack2<kBf16>(v[8 * j + 2], v[8 * j + 3]);
            q.z = pack2<kBf16>(v[8 * j + 4], v[8 * j + 5]);
            q.w = pack2<kBf16>(v[8 * j + 6], v[8 * j + 7]);
            *reinterpret_cast<uint4*>(box + lane * 64u + ((j ^ ((lane >> 1) & 3u)) << 4)) = q;
        }
    }
    __device__ __forceinline__ void send(const CUtensorMap* map, const uint8_t* box, int col, int row) const {
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(map, box, col, row);
            bulk_commit_group();
        }
    }

    template <bool kBf16>
    __device__ __forceinline__ void put16(const CUtensorMap* map, const float (&v)[32], int col, int row) {
        uint8_t* box = take();
        fill<kBf16>(box, v);
        send(map, box, col, row);
    }

    // Two boxes (the second one with `two`) with one hand-over to the stores.
    template <bool kBf16>
    __device__ __forceinline__ void put16_two(const CUtensorMap* map, const float (&v)[32], const float (&w)[32],
                                              bool two, int col, int col_two, int row) {
        whole = true;
        if (lane == 0) bulk_wait_group_read<0>();
        __syncwarp();
        fill<kBf16>(bufs, v);
        if (two) fill<kBf16>(bufs + kTrainBoxBytes, w);
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(map, bufs, col, row);
            if (two) tma_store_2d(map, bufs + kTrainBoxBytes, col_two, row);
            bulk_commit_group();
        }
    }

    // This lane's row of a box.
    __device__ __forceinline__ Row32 row_of(const uint8_t* box) const {
        Row32 r;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            r.w[j] = *reinterpret_cast<const uint4*>(box + lane * 64u + ((j ^ ((lane >> 1) & 3u)) << 4));
        return r;
    }

    // The transposed box: lane = column `col` + lane, v = rows row .. row + 31.
    template <bool kBf16>
    __device__ __forceinline__ void put16_turned(const CUtensorMap* map, const float (&v)[32], int col, int row) {
        uint8_t* box = take();
#pragma unroll
        for (uint32_t i = 0; i < 32; i += 2) {
            const uint32_t w = pack2<kBf16>(v[i], v[i + 1]);
            const uint32_t at = (((lane >> 3) ^ ((i >> 1) & 3u)) << 4) + (lane & 7u) * 2u;   // alike for i and i + 1
            *reinterpret_cast<uint16_t*>(box + i * 64u + at) = static_cast<uint16_t>(w);
            *reinterpret_cast<uint16_t*>(box + i * 64u + 64u + at) = static_cast<uint16_t>(w >> 16);
        }
        send(map, box, col, row);
    }

    __device__ void put32(const CUtensorMap* map, const float (&v)[32], bool add, int col, int row) {
        whole = true;
        if (lane == 0) bulk_wait_group_read<0>();
        __syncwarp();
        uint8_t* box = bufs;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(box + lane * 128u + ((j ^ (lane & 7u)) << 4)) =
                make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
            if (add)
                tma_reduce_add_2d(map, box, col, row);
            else
                tma_store_2d(map, box, col, row);
            bulk_commit_group();
        }
    }
};

// Two accumulator groups, loaded together.
__device__ __forceinline__ void tmem_ld32_two(uint32_t t, uint32_t t_two, float (&v)[32], float (&w)[32]) {
    uint32_t a[32], b[32];
    tmem_ld_32x32b_x32(t, a);
    tmem_ld_32x32b_x32(t_two, b);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        v[i] = __uint_as_float(a[i]);
        w[i] = __uint_as_float(b[i]);
    }
}

__device__ __forceinline__ void tmem_ld32(uint32_t t, float (&v)[32]) {
    uint32_t r[32];
    tmem_ld_32x32b_x32(t, r);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Row and column of a problem's tile t: grouped raster order, or the upper
// triangle row by row.
__device__ __forceinline__ void tile_place(int t, int tiles_m, int tiles_n, int group_m, int symmetric, int& tm, int& tn) {
    if (!symmetric) {
        tile_coords(t, tiles_m, tiles_n, group_m, tm, tn);
        return;
    }
    tm = 0;
    for (int left = tiles_n; t >= left; --left) {
        t -= left;
        ++tm;
    }
    tn = tm + t;
}
__device__ __forceinline__ void tile_place(const TrainProblem& q, int t, int& tm, int& tn) {
    tile_place(t, q.tiles_m, q.tiles_n, q.group_m, q.symmetric, tm, tn);
}

// The tiles of one unit (CTA or pair) in order; every role iterates alike.
// Problem 0's tiles ("heavy": the longest sums) go round robin; where they do
// not divide evenly the units that took one more sit out the first
// `light_skip` waves of the other problems' tiles, which are shorter.
struct TileIter {
    int unit, units, next_heavy, wave;
    int prob, tm, tn;      // the current tile
    int local;             // its number among the problem's
    int split, kb0, kb1;   // its part of the sum: K blocks [kb0, kb1)
    bool back;             // walk K from the end
    __device__ TileIter(int u, int n) : unit(u), units(n), next_heavy(u), wave(0) {}
    __device__ bool next(const TrainParams& p) {
        int t, nth;
        if (next_heavy < p.heavy_tiles) {
            prob = 0;
            t = next_heavy;
            nth = next_heavy / units;
            next_heavy += units;
        } else {
            const int rest = p.heavy_tiles % units;
            if (wave < p.light_skip && unit < rest) wave = p.light_skip;
            t = wave < p.light_skip ? wave * (units - rest) + unit - rest
                                    : p.light_skip * (units - rest) + (wave - p.light_skip) * units + unit;
            nth = wave;
            ++wave;
            if (t >= p.light_tiles) return false;
            prob = 1;
            while (t >= p.prob[prob].tiles * p.prob[prob].splits) {
                t -= p.prob[prob].tiles * p.prob[prob].splits;
                ++prob;
            }
        }
        const TrainProblem& q = p.prob[prob];
        split = q.splits > 1 ? t / q.tiles : 0;
        local = t - split * q.tiles;
        tile_place(q, q.tile0 + local, tm, tn);
        kb0 = split * q.kb_split;
        kb1 = min(q.nkb, kb0 + q.kb_split);
        // Odd waves walk K backwards: they start on the panels that the wave
        // before read last, while those are in L2.
        back = (nth & 1) != 0;
        return true;
    }
    // K blocks [from, to) of segment 0 or 1 in this part.
    __device__ void segment(const TrainProblem& q, int seg, int& from, int& to) const {
        from = seg ? max(kb0 - q.nkb0, 0) : min(kb0, q.nkb0);
        to = seg ? max(kb1 - q.nkb0, 0) : min(kb1, q.nkb0);
    }
};

// ---------------------------------------------------------------- epilogues ---

// One epilogue warp's part of a tile: rows row0 + lane, the groups of 32 columns
// with index group, group + 2, ... of tile column tn. begin() starts loads before
// the accumulator is ready (C of all groups: a x X + poly X of 1024 x 2560 took
// 2.8 us of epilogue with a group ahead); run() goes through the groups. Called
// by the whole warp.
template <int kEpi>
struct TrainEpilogue {
    const TrainParams& p;
    const TrainProblem& q;
    int row0, row, tn, width, first;   // width: the tile's output columns
    int out_row, mirror;               // row0 in the output; the tile is stored transposed too
    bool in_rows;
    int out_kind, out_bf16;
    float alpha, beta;
    const float* alpha_ptr;
    const void* c0;
    long long ldc;
    Row32 x[kEpi == kTrainStoreC ? 4 : 1];         // C of all groups of the tile
    Patch32 silu, slope;                           // kTrainGateGrad: what was kept, of one group
    uint32_t lane_;

    // in_tile: this warp's first row in the tile.
    __device__ TrainEpilogue(const TrainParams& p_, const TrainProblem& q_, const TileIter& it, int tile_m, int in_tile,
                             int lane, int group)
        : p(p_), q(q_), row0(it.tm * tile_m + in_tile), row(row0 + lane), tn(it.tn),
          width(kEpi == kTrainGate ? q_.tile_n / 2 : q_.tile_n), first(32 * group),
          out_row(q_.parted ? (it.split * q_.tiles + it.local) * tile_m + in_tile : row0),
          mirror(q_.symmetric && it.tn > it.tm), in_rows(row < q_.m), out_kind(q_.out_kind), out_bf16(p_.out_bf16),
          alpha(q_.alpha), beta(q_.beta), alpha_ptr(q_.alpha_ptr), c0(q_.c), ldc(q_.ldc),
          lane_(static_cast<uint32_t>(lane)) {}

    __device__ __forceinline__ void fetch(int c) {
        const int col = tn * width + c, cols = c < width ? q.n - col : 0;
        silu.load(p.silu, p.ld_kept, row0, col, q.m - row0, cols, lane_);
        slope.load(p.slope, p.ld_kept, row0, col, q.m - row0, cols, lane_);
    }
    // What was kept comes from DRAM: one 128-byte line per row and 64 columns into
    // L2 while the tile is still multiplied, or each group's loads would wait for
    // memory in turn.
    __device__ void begin() {
        if constexpr (kEpi == kTrainGateGrad) {
            const void* src = first == 0 ? p.silu : p.slope;
            for (int c = 0; c < width && in_rows && tn * width + c < q.n; c += 64)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint16_t*>(src) + row * p.ld_kept + tn * width + c));
            fetch(first);
        }
        if constexpr (kEpi == kTrainStoreC) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = first + 64 * k, col = tn * width + c;
                x[k].load(c0, row * ldc + col, in_rows && c < width ? q.n - col : 0);
            }
        }
    }

    // t: TMEM address of the accumulator, this warp's lane quarter. The output
    // type is a template parameter: choosing it per pair of elements doubled the
    // instructions, and with two epilogue warps a scheduler these set the time
    // of tiles with short sums.
    __device__ __forceinline__ void run(BoxWriter& box, uint32_t t) {
        if (row0 >= q.m) return;
        if constexpr (kEpi == kTrainLse) {
            statistics(t);
        } else if ((kEpi == kTrainStore || kEpi == kTrainStoreC) && out_kind != kTrainOut16) {
#pragma unroll 1
            for (int c = first; c < width && tn * width + c < q.n; c += 64) {
                float v[32];
                tmem_ld32(t + c, v);
                box.put32(&q.out[0], v, out_kind == kTrainOutF32Add, c, out_row);
            }
        } else if (out_bf16) {
            store<true>(box, t);
        } else {
            store<false>(box, t);
        }
    }

    // Running maximum and sum over this thread's columns of the tile, four
    // interleaved chains of each.
    __device__ __forceinline__ void statistics(uint32_t t) {
        const float kNone = __int_as_float(0xff800000);
        const long long want = in_rows ? p.target[row] - p.col_base : -1;
        float top = kNone, sum = 0.f;
#pragma unroll 1
        for (int c = first; c < width; c += 64) {
            const int col = tn * width + c;
            if (col >= q.n) break;
            float v[32];
            tmem_ld32(t + c, v);
            if (want >= col && want < col + 32 && want < q.n) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (col + i == want) p.target_logit[row] = v[i];
            }
            if (col + 32 > q.n) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (col + i >= q.n) v[i] = kNone;
            }
            float best[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
            for (int i = 4; i < 32; ++i) best[i & 3] = fmaxf(best[i & 3], v[i]);
            const float most = fmaxf(fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3])), top);
            // No column above -inf yet: subtract 0, so that exp gives 0, not NaN.
            const float ref = most == kNone ? 0.f : most;
            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 32; ++i) part[i & 3] += exp2_fast((v[i] - ref) * kLog2e);
            sum = fmaf(sum, exp2_fast((top - ref) * kLog2e), (part[0] + part[1]) + (part[2] + part[3]));
            top = most;
        }
        if (in_rows) p.partial[static_cast<long long>(2 * tn + first / 32) * q.m + row] = make_float2(top, sum);
    }

    template <bool kBf16>
    __device__ __forceinline__ void store(BoxWriter& box, uint32_t t) {
        float scale = 0.f, lse = 0.f, ratio = 0.f;
        long long want = -1;
        if constexpr (kEpi == kTrainStore || kEpi == kTrainStoreC)
            if (alpha_ptr != nullptr) alpha *= *alpha_ptr;
        if constexpr (kEpi == kTrainStore)
            if (q.alpha_rows != nullptr && in_rows) alpha *= q.alpha_rows[row];
        if constexpr (kEpi == kTrainLogitGrad)
            if (in_rows) {
                want = p.target[row] - p.col_base;
                scale = p.row_scale[row];
                lse = p.lse[row];
                if (p.row_ratio != nullptr) ratio = p.row_ratio[row];
            }
        if (kEpi == kTrainLogitGrad || (kEpi == kTrainStore && !mirror)) {
            // Two groups a turn.
#pragma unroll 1
            for (int c = first; c < width; c += 128) {
                const int col = tn * width + c;
                if (col >= q.n) break;
                const bool two = c + 64 < width && col + 64 < q.n;
                float v[32], w[32];
                tmem_ld32_two(t + c, two ? t + c + 64 : t + c, v, w);
                if constexpr (kEpi == kTrainStore) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        v[i] *= alpha;
                        w[i] *= alpha;
                    }
                } else {
                    logit_gradient(v, col, want, scale, lse);
                    logit_gradient(w, col + 64, want, scale, lse);
                }
                box.put16_two<kBf16>(&q.out[0], v, w, two, col, col + 64, row0);
                if constexpr (kEpi == kTrainLogitGrad) {
                    if (p.row_ratio != nullptr) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            v[i] *= ratio;
                            w[i] *= ratio;
                        }
                        box.put16_two<kBf16>(&q.out[1], v, w, two, col, col + 64, row0);
                    }
                }
            }
            return;
        }
        if constexpr (kEpi == kTrainStoreC) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = first + 64 * k, col = tn * width + c;
                if (c >= width || col >= q.n) break;
                float v[32];
                tmem_ld32(t + c, v);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 w = x[k].template pair<false>(i);   // C is FP16
                    v[2 * i] = fmaf(alpha, v[2 * i], beta * w.x);
                    v[2 * i + 1] = fmaf(alpha, v[2 * i + 1], beta * w.y);
                }
                box.put16<kBf16>(&q.out[0], v, col, row0);
                if (mirror) box.put16_turned<kBf16>(&q.out[0], v, row0, col);
            }
            return;
        }
#pragma unroll 1
        for (int c = first; c < width; c += 64) {
            const int col = tn * width + c;
            if (col >= q.n) break;
            float v[32];
            if constexpr (kEpi == kTrainStore) {
                tmem_ld32(t + c, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] *= alpha;
                box.put16<kBf16>(&q.out[0], v, col, row0);
                box.put16_turned<kBf16>(&q.out[0], v, row0, col);
            } else if constexpr (kEpi == kTrainGate) {
                float u[32];
                tmem_ld32(t + c, v);
                tmem_ld32(t + width + c, u);
                if (p.keep) {
                    float d[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float s = sigmoid_f(v[i]);
                        v[i] *= s;
                        // silu' = s (1 + g (1 - s)) = s + silu (1 - s)
                        d[i] = u[i] * fmaf(v[i], 1.f - s, s);
                        u[i] *= v[i];
                    }
                    box.put16<kBf16>(&q.out[0], u, col, row0);
                    box.put16<kBf16>(&q.out[1], v, col, row0);
                    box.put16<kBf16>(&q.out[2], d, col, row0);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) u[i] *= v[i] * sigmoid_f(v[i]);
                    box.put16<kBf16>(&q.out[0], u, col, row0);
                }
            } else if constexpr (kEpi == kTrainGateGrad) {
                // The patches of this group through the two boxes to their rows'
                // lanes, and the results into the same places.
                uint8_t* other = box.bufs + kTrainBoxBytes;
                if (box.lane == 0) bulk_wait_group_read<0>();
                __syncwarp();
                silu.put(box.bufs, box.lane);
                slope.put(other, box.lane);
                fetch(c + 64);
                __syncwarp();
                const Row32 s = box.row_of(box.bufs), d = box.row_of(other);
                tmem_ld32(t + c, v);
                float du[32];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 si = s.template pair<kBf16>(i), di = d.template pair<kBf16>(i);
                    du[2 * i] = v[2 * i] * si.x;
                    du[2 * i + 1] = v[2 * i + 1] * si.y;
                    v[2 * i] *= di.x;
                    v[2 * i + 1] *= di.y;
                }
                box.fill<kBf16>(box.bufs, v);
                box.fill<kBf16>(other, du);
                fence_async_shared();
                __syncwarp();
                if (box.lane == 0) {
                    tma_store_2d(&q.out[0], box.bufs, col, row0);
                    tma_store_2d(&q.out[1], other, col, row0);
                    bulk_commit_group();
                }
            }
        }
    }

    // (exp(z - lse) - [column == target]) scale. A row without a target has factor
    // 0 and gradient 0, whatever its logits.
    __device__ __forceinline__ void logit_gradient(float (&v)[32], int col, long long want, float scale, float lse) const {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = scale == 0.f ? 0.f : exp2_fast((v[i] - lse) * kLog2e) * scale;
        if (want >= col && want < col + 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (col + i == want) v[i] -= scale;
        }
    }
};

// ------------------------------------------------------------------ the GEMM ---

// 1 in one lane of the (converged) warp, 0 in the others.
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}

// tcgen05.mma and commit by the lane with `issuer` set; called by the whole warp.
template <bool kPair>
__device__ __forceinline__ void tc_mma_if(uint32_t issuer, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                          uint32_t idesc, uint32_t accumulate) {
    if constexpr (kPair)
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                     "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(issuer) : "memory");
    else
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                     "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(issuer) : "memory");
}
template <bool kPair>
__device__ __forceinline__ void tc_commit_if(uint32_t issuer, uint32_t bar) {
    if constexpr (kPair)   // the barrier at the same place in both CTAs
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
                     "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
                     " [%0], %1;\n\t}" ::"r"(bar), "h"(static_cast<uint16_t>(0x3)), "r"(issuer) : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                     "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                     ::"r"(bar), "r"(issuer) : "memory");
}

// Frees an accumulator: arrives at the leader CTA's barrier (shared::cluster
// address). Ordered after this warp's TMEM reads by tcgen05.wait::ld and the
// fence before; no other memory is handed over, so no cluster-wide release,
// which waits for the tile's stores on their way (900 to 3000 cycles a tile).
__device__ __forceinline__ void acc_release_pair(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// A compile-time argument of the producer's inner loop, and the ways B comes.
template <int kValue>
struct Is {
    static constexpr int value = kValue;
};
enum : int { kBKMajor = 0, kBMnMajor = 1, kBTwoHalves = 2 };

template <bool kPair, int kEpi>
__global__ void __launch_bounds__(kTrainThreads, 1) train_gemm_kernel(const __grid_constant__ TrainParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align_1024(smem_raw);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kTrainDataBytes);   // pair: the even CTA's
    uint64_t* empty = full + kTrainMaxStages;
    uint64_t* tfull = empty + kTrainMaxStages;   // [2]
    uint64_t* tempty = tfull + 2;                // [2], pair: the even CTA's
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    constexpr int kTileM = kPair ? 256 : 128;
    const uint32_t warp = warp_index();
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t rank = kPair ? cluster_ctarank() : 0u;
    const bool leader = rank == 0;

    if (warp == kTrainEpiWarps && lane == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1u);
            mbar_init(&empty[s], 1u);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&tfull[i], 1u);
            mbar_init(&tempty[i], (kPair ? 2u : 1u) * kTrainEpiWarps);   // one lane of each epilogue warp
        }
        mbar_init(drain, 1u);
        *abort_flag = 0;
        mbar_init_fence();
        tma_prefetch_map(&p.prob[0].a[0]);
        tma_prefetch_map(&p.prob[0].b[0]);
        if constexpr (kEpi == kTrainGate) tma_prefetch_map(&p.prob[0].b[1]);
        if constexpr (kEpi != kTrainLse) tma_prefetch_map(&p.prob[0].out[0]);
    }
    if (warp == kTrainEpiWarps + 1) {
        if constexpr (kPair) {
            tmem_alloc_pair(tmem_slot, 2 * kTrainAccCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, 2 * kTrainAccCols);
            tmem_relinquish();
        }
    }
    tc_fence_before_sync();
    if constexpr (kPair) cluster_sync();         // both CTAs' barriers exist before any remote op
    else __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    grid_dependents_launch();
    // Every role looks its first tile up before it waits for the previous
    // kernel: the parameters come cold from constant memory, about 1.1 us of
    // misses one after the other, which that kernel's end then hides.
    const WaitCtl wc{abort_flag, p.status, p.timeout_ns};
    const int unit = kPair ? blockIdx.x >> 1 : blockIdx.x;
    const int units = kPair ? gridDim.x >> 1 : gridDim.x;
    TileIter it(unit, units);

    const uint32_t num_stages = static_cast<uint32_t>(p.stages), block_stride = p.block_stride;
    const int sub = p.sub;
    const uint32_t stage_bytes = static_cast<uint32_t>(sub) * block_stride, b_offset = p.b_offset;
    const uint32_t ring = smem_addr(smem);

    if (warp == kTrainEpiWarps) {
        if (lane == 0) {
            uint32_t stage = 0, phase = 0, issued = 0;
            bool ok = true;
            // Everything the inner loop needs is in registers: parameter loads
            // between the copies cost 15-30 % of a 256 x 256 tile's K block.
            const uint32_t full0 = kPair ? map_to_rank(smem_addr(full), 0) : smem_addr(full);
            auto load = [](uint32_t dst, uint64_t map, uint32_t bar, int x, int y) {
                if constexpr (kPair)
                    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global"
                                 ".mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
                else
                    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
                                 " [%0], [%1, {%3, %4}], [%2];"
                                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
            };
            auto map_of = [](const CUtensorMap& m) { return reinterpret_cast<uint64_t>(&m); };
            uint32_t extra = p.inject ? 16u : 0u;
            bool waiting = true;   // for the previous kernel
            // The K blocks of one segment, forwards or backwards, two to a stage.
            auto segment = [&](uint64_t ma, uint64_t mb, uint64_t mb2, auto a_mn_c, auto b_kind_c, int row0, int col0,
                               int chunks, uint32_t half_bytes, uint32_t block_bytes, int from, int to, bool back) {
                constexpr bool a_mn = decltype(a_mn_c)::value;
                constexpr int b_kind = decltype(b_kind_c)::value;
                int k = (back ? to - 1 : from) * kBlockK;
                const int step = back ? -kBlockK : kBlockK;
                if (waiting) grid_dependency_wait();
                waiting = false;
                for (int left = to - from; left > 0; left -= sub) {
                    if (!(kPair ? mbar_wait_cluster(&empty[stage], phase ^ 1u, wc)
                                : mbar_wait(&empty[stage], phase ^ 1u, wc))) return false;
                    const int count = left < sub ? left : sub;
                    if (leader) mbar_arrive_expect_tx(&full[stage], (kPair ? 2u : 1u) * count * block_bytes + extra);
                    extra = 0;
                    const uint32_t bar = full0 + stage * 8u;
                    uint32_t s_a = ring + stage * stage_bytes;
                    for (int i = 0; i < count; ++i, s_a += block_stride, k += step) {
                        const uint32_t s_b = s_a + b_offset;
                        if constexpr (a_mn) {
                            load(s_a, ma, bar, row0, k);
                            load(s_a + kChunkBytes, ma, bar, row0 + 64, k);
                        } else {
                            load(s_a, ma, bar, k, row0);
                        }
                        if constexpr (b_kind == kBMnMajor) {
                            load(s_b, mb, bar, col0, k);
                            if (chunks > 1) load(s_b + kChunkBytes, mb, bar, col0 + 64, k);
                            if (!kPair && chunks > 2) load(s_b + 2 * kChunkBytes, mb, bar, col0 + 128, k);
                            if (!kPair && chunks > 3) load(s_b + 3 * kChunkBytes, mb, bar, col0 + 192, k);
                        } else {
                            load(s_b, mb, bar, k, col0);
                            if constexpr (b_kind == kBTwoHalves) load(s_b + half_bytes, mb2, bar, k, col0);
                        }
                    }
                    ++issued;
                    if (++stage == num_stages) { stage = 0; phase ^= 1u; }
                }
                return true;
            };
            while (ok && it.next(p)) {
                const TrainProblem& q = p.prob[it.prob];
                const int row0 = it.tm * kTileM + static_cast<int>(rank) * 128;
                // Columns of B that this CTA loads: all, or its half of the pair's.
                const int cols = kPair ? q.tile_n / 2 : q.tile_n;
                const bool dual = kEpi == kTrainGate, back = it.back;
                const int col0 = dual ? it.tn * (q.tile_n / 2) : it.tn * q.tile_n + static_cast<int>(rank) * cols;
                const int chunks = (cols + 63) / 64;
                const uint32_t bytes = q.a_tile_bytes + (q.b_mn ? chunks * kChunkBytes : cols * 128u);
                for (int i = 0; i < 2 && ok; ++i) {
                    const int seg = back ? 1 - i : i;
                    int from, to;
                    it.segment(q, seg, from, to);
                    if (from >= to) continue;
                    const uint64_t ma = map_of(q.a[seg]), mb = map_of(q.b[seg]);
                    if constexpr (dual) {
                        if constexpr (kPair)
                            ok = segment(ma, map_of(q.b[rank]), 0ull, Is<0>{}, Is<kBKMajor>{}, row0, col0, chunks, 0u,
                                         bytes, from, to, back);
                        else
                            ok = segment(ma, mb, map_of(q.b[1]), Is<0>{}, Is<kBTwoHalves>{}, row0, col0, chunks,
                                         cols * 64u, bytes, from, to, back);
                    } else if (q.a_mn) {
                        ok = q.b_mn ? segment(ma, mb, 0ull, Is<1>{}, Is<kBMnMajor>{}, row0, col0, chunks, 0u, bytes,
                                              from, to, back)
                                    : segment(ma, mb, 0ull, Is<1>{}, Is<kBKMajor>{}, row0, col0, chunks, 0u, bytes,
                                              from, to, back);
                    } else {
                        ok = q.b_mn ? segment(ma, mb, 0ull, Is<0>{}, Is<kBMnMajor>{}, row0, col0, chunks, 0u, bytes,
                                              from, to, back)
                                    : segment(ma, mb, 0ull, Is<0>{}, Is<kBKMajor>{}, row0, col0, chunks, 0u, bytes,
                                              from, to, back);
                    }
                }
            }
            if (leader && (!ok || *abort_flag)) {
                // In-flight copies land before the CTA (or its pair) leaves.
                for (uint32_t s = 0; s < (issued < num_stages ? issued : num_stages); ++s) {
                    const uint32_t arms = issued / num_stages + (s < issued % num_stages ? 1u : 0u);
                    mbar_wait_drain(&full[s], (arms - 1u) & 1u, kDrainLimitNs);
                }
            }
        }
    } else if (warp == kTrainEpiWarps + 1) {
        if (leader) {
            // The whole warp walks the loop and one elected lane issues: with
            // warp-uniform control flow the descriptors stay in uniform
            // registers, where one lane alone pays a move per operand and MMA.
            const uint32_t issuer = elect_lane();
            uint32_t stage = 0, phase = 0, iter = 0;
            bool ok = true;
            const uint32_t format = p.in_bf16 ? (1u << 7) | (1u << 10) : 0u;
            while (ok && it.next(p)) {
                const TrainProblem& q = p.prob[it.prob];
                const uint32_t idesc = make_idesc_f16(kTileM, 0, q.a_mn, q.b_mn) | format |
                                       (static_cast<uint32_t>(q.tile_n >> 3) << 17);
                // 16 of K further: 32 bytes along a K-major row, 16 rows of 128 bytes MN-major.
                const uint64_t step_a = q.a_mn ? 2048u >> 4 : 32u >> 4;
                const uint64_t step_b = q.b_mn ? 2048u >> 4 : 32u >> 4;
                const uint64_t desc_a = make_smem_desc(ring, q.a_mn ? kChunkBytes : 16u, 1024u);
                const uint64_t desc_b = make_smem_desc(ring + b_offset, q.b_mn ? kChunkBytes : 16u, 1024u);
                const uint32_t acc = iter & 1u, acc_phase = (iter >> 1) & 1u;
                if (iter++ == 0) grid_dependency_wait();   // the time limits of waits start then
                if (!__all_sync(0xffffffffu, kPair ? mbar_wait_cluster(&tempty[acc], acc_phase ^ 1u, wc)
                                                   : mbar_wait(&tempty[acc], acc_phase ^ 1u, wc))) { ok = false; break; }
                tc_fence_after_sync();
                const uint32_t d = tmem_base + acc * kTrainAccCols;
                uint32_t add = 0;
                auto block = [&](uint64_t off) {
                    const uint64_t da = desc_a + off, db = desc_b + off;
#pragma unroll
                    for (int kk = 0; kk < kBlockK / 16; ++kk) {
                        tc_mma_if<kPair>(issuer, d, da + kk * step_a, db + kk * step_b, idesc, add);
                        add = 1;
                    }
                };
                for (int i = 0; i < 2 && ok; ++i) {
                    int from, to;
                    it.segment(q, it.back ? 1 - i : i, from, to);
                    for (int left = to - from; left > 0; left -= sub) {
                        if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, wc))) { ok = false; break; }
                        const uint64_t off = (stage * stage_bytes) >> 4;
                        block(off);
                        if (sub > 1 && left > 1) block(off + (block_stride >> 4));
                        tc_commit_if<kPair>(issuer, smem_addr(&empty[stage]));
                        if (++stage == num_stages) { stage = 0; phase ^= 1u; }
                    }
                }
                if (ok) tc_commit_if<kPair>(issuer, smem_addr(&tfull[acc]));
            }
            if (!ok && issuer) {
                if constexpr (kPair) tc_commit_pair(smem_addr(drain));
                else tc_commit(drain);
                mbar_wait_drain(drain, 0, kDrainLimitNs);
            }
        }
    } else {
        const uint32_t tempty0 = kPair ? map_to_rank(smem_addr(&tempty[0]), 0) : 0u;
        const uint32_t tempty1 = kPair ? map_to_rank(smem_addr(&tempty[1]), 0) : 0u;
        BoxWriter box{smem + kTrainRingBytes + warp * 2u * kTrainBoxBytes, 0u, lane, false};
        const int quarter = static_cast<int>(warp & 3u), group = static_cast<int>(warp >> 2);
        uint32_t iter = 0;
        while (it.next(p)) {
            const uint32_t acc = iter & 1u, acc_phase = (iter >> 1) & 1u;
            ++iter;
            TrainEpilogue<kEpi> epi(p, p.prob[it.prob], it, kTileM, static_cast<int>(rank) * 128 + quarter * 32,
                                    static_cast<int>(lane), group);
            if (iter == 1) grid_dependency_wait();
            epi.begin();
            const bool got = kPair ? mbar_wait_cluster(&tfull[acc], acc_phase, wc) : mbar_wait(&tfull[acc], acc_phase, wc);
            if (!__all_sync(0xffffffffu, got)) break;
            tc_fence_after_sync();
            epi.run(box, tmem_base + ((quarter * 32u) << 16) + acc * kTrainAccCols);
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (kPair) acc_release_pair(acc ? tempty1 : tempty0);
                else mbar_arrive(&tempty[acc]);
            }
        }
        if (lane == 0) bulk_wait_group_all();
    }

    __syncwarp();
    if (kPair && *abort_flag) settle_ns(2000000ull);   // the peer's copies towards this CTA land
    tc_fence_before_sync();
    if constexpr (kPair) cluster_sync();               // no CTA leaves while its pair may still touch it
    else __syncthreads();
    if (warp == kTrainEpiWarps + 1) {
        tc_fence_after_sync();
        if constexpr (kPair) tmem_dealloc_pair(tmem_base, 2 * kTrainAccCols);
        else tmem_dealloc(tmem_base, 2 * kTrainAccCols);
    }
}

// -------------------------------------------------- cross entropy, row parts ---

// Factor on the stored logit gradients of one incoming gradient, so that a
// probability of 1 / vocabulary stays a normal FP16 number (151936 entries:
// 0.1); the products' epilogues take it out again.
constexpr float kLogitGradScale = 16384.f;

// Joins a row's per-tile (max, sum) pairs: lse = max + log(sum), and its loss
// lse - logit[target], formed as (max - logit) + log(sum). A row whose target
// is `ignore` has loss 0; one outside the vocabulary gets NaN.
// Block (kRows rows, 1024 / kRows slices of the pairs), joined in shared memory;
// a thread has four pairs in flight. 8 rows to a block: with 32 there are few
// blocks and a thread walks many pairs in turn (182 rows x 126940: 14 us).
__device__ __forceinline__ float2 join_pairs(float2 a, float2 b) {
    const float best = fmaxf(a.x, b.x);
    const float ref = best == __int_as_float(0xff800000) ? 0.f : best;
    // A NaN sum stays NaN.
    return make_float2(best, a.y * exp2_fast((a.x - ref) * kLog2e) + b.y * exp2_fast((b.x - ref) * kLog2e));
}

template <int kRows>
__global__ void __launch_bounds__(1024) lse_join_kernel(const float2* partial, int tiles, int m,
                                                        const float* target_logit,
                                                        const long long* target, long long vocab,
                                                        long long ignore, float* lse,
                                                        float* loss) {
    constexpr int kSlices = 1024 / kRows;
    __shared__ float2 part[kSlices][kRows + 1];
    grid_dependents_launch();
    grid_dependency_wait();
    const int row = blockIdx.x * kRows + threadIdx.x;
    const float2 none = make_float2(__int_as_float(0xff800000), 0.f);
    float2 all = none;
    if (row < m)
        for (int t = threadIdx.y; t < tiles; t += 4 * kSlices) {
            float2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = t + kSlices * i;
                v[i] = at < tiles ? partial[static_cast<long long>(at) * m + row] : none;
            }
            all = join_pairs(all, join_pairs(join_pairs(v[0], v[1]), join_pairs(v[2], v[3])));
        }
    part[threadIdx.y][threadIdx.x] = all;
    __syncthreads();
    for (int half = kSlices / 2; half > 0; half /= 2) {
        if (static_cast<int>(threadIdx.y) < half)
            part[threadIdx.y][threadIdx.x] =
                join_pairs(part[threadIdx.y][threadIdx.x], part[threadIdx.y + half][threadIdx.x]);
        __syncthreads();
    }
    if (threadIdx.y != 0 || row >= m) return;
    all = part[0][threadIdx.x];
    const float ls = logf(all.y);
    lse[row] = all.x + ls;
    const long long want = target[row];
    if (want == ignore) loss[row] = 0.f;
    else loss[row] = (want >= 0 && want < vocab) ? (all.x - target_logit[row]) + ls : __int_as_float(0x7fffffff);
}

// Sum of the rows' losses (and their count for the mean), one block, in a
// fixed order and 64 bits. Latency: 3.6-4.5 us for 24 to 4096 rows.
__global__ void __launch_bounds__(1024) loss_reduce_kernel(const float* loss,
                                                           const long long* target, int m,
                                                           long long ignore, int mean, float* out) {
    __shared__ double sums[32];
    __shared__ int counts[32];
    grid_dependents_launch();
    grid_dependency_wait();
    double s = 0.;
    int c = 0;
    for (int i = threadIdx.x; i < m; i += 1024) {
        s += static_cast<double>(loss[i]);
        c += target[i] != ignore;
    }
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        c += __shfl_xor_sync(0xffffffffu, c, o);
    }
    if ((threadIdx.x & 31) == 0) {
        sums[threadIdx.x >> 5] = s;
        counts[threadIdx.x >> 5] = c;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < 32; ++i) {
        s += sums[i];
        c += counts[i];
    }
    *out = static_cast<float>(mean ? s / c : s);   // no target at all: 0 / 0 = NaN for the mean
}

// Row factors of the logits' gradient, and what takes them out of the products:
//   dz[row] = row_scale[row] (p - onehot), dW = alpha dz^T x, dx = alpha dz W.
// One incoming gradient for all rows: row_scale is 2^14 and alpha has the rest.
// Infinity and NaN go to the rows they belong to, where alpha would bring them
// to the others (0 x inf); an ignored row's gradient is 0 in any case.
// One per row, kScaleBf16: row_scale = dloss[row] 2^k, alpha = 2^-k, with the
// largest at 2^60 (k at most 100, which FP32 has the inverse of): BF16's range
// then holds probabilities in rows with 1e-40 of it. FP16 with one scale for all rows loses probabilities of small
// gradients: 1/151936 is subnormal in a row with 1/1800 of the largest, and zero
// with 1/3.6e6. A sum over rows (dW) needs one scale, a row of dx does not, so dz
// is written in both where both are wanted. kScaleRows: row_scale = dloss[row]
// 2^(15 - e), e the row's own exponent, and dx = row_alpha[row] dz W; row_ratio =
// 2^(e - E), E the largest exponent, turns such a dz into the common scale's.
// kScaleCommon: that scale alone, dloss[row] 2^(15 - E); alpha = 2^(E - 15).
// Block 0; latency, 4.6-5.9 us for 24 to 4096 rows. Further blocks, where dW is
// wanted, copy x with zeros for the ignored rows: their dz is 0, but dz^T x would
// still take infinity and NaN from them (padding may hold anything). With the copy
// 6-7 us at 777 x 1024, 11-13 us at 4096 x 2560 (42 MB, cold).
enum : int { kScaleOne = 0, kScaleBf16 = 1, kScaleCommon = 2, kScaleRows = 3 };
__global__ void __launch_bounds__(1024) logit_grad_setup_kernel(const float* dloss, int kind, int mean,
                                                                const long long* target, int m,
                                                                long long vocab, long long ignore,
                                                                float* row_scale, float* row_alpha,
                                                                float* row_ratio, float* alpha, const void* x,
                                                                long long ldx, int hidden, void* x_kept) {
    __shared__ float tops[32];
    __shared__ int counts[32];
    grid_dependents_launch();
    grid_dependency_wait();
    if (blockIdx.x > 0) {
        const int per_row = hidden / 8;
        const long long total = static_cast<long long>(m) * per_row, stride = (gridDim.x - 1) * 1024ll;
#pragma unroll 4
        for (long long i = (blockIdx.x - 1) * 1024ll + threadIdx.x; i < total; i += stride) {
            const long long r = i / per_row;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (target[r] != ignore)
                v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + r * ldx + (i - r * per_row) * 8);
            static_cast<uint4*>(x_kept)[i] = v;
        }
        return;
    }
    const float kMost = 3.4028235e38f;   // the largest finite number
    const bool one_finite = kind == kScaleOne && fabsf(dloss[0]) <= kMost;
    float top = 0.f;                      // of the finite ones
    int c = 0;
    for (int i = threadIdx.x; i < m; i += 1024) {
        if (target[i] == ignore) continue;
        ++c;
        if (kind != kScaleOne) {
            const float a = fabsf(dloss[i]);
            if (a <= kMost) top = fmaxf(top, a);
        }
    }
    for (int o = 16; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        c += __shfl_xor_sync(0xffffffffu, c, o);
    }
    if ((threadIdx.x & 31) == 0) {
        tops[threadIdx.x >> 5] = top;
        counts[threadIdx.x >> 5] = c;
    }
    __syncthreads();
    top = 0.f;
    c = 0;
    for (int i = 0; i < 32; ++i) {
        top = fmaxf(top, tops[i]);
        c += counts[i];
    }
    int most = 0;
    if (top > 0.f) frexpf(top, &most);
    const int up = min(60 - most, 100);   // kScaleBf16
    const float nan = __int_as_float(0x7fffffff);
    for (int i = threadIdx.x; i < m; i += 1024) {
        const long long want = target[i];
        float r = 0.f, own_alpha = 1.f, ratio = 1.f;
        if (want != ignore) {
            const float d = kind == kScaleOne ? dloss[0] : dloss[i];
            r = one_finite ? kLogitGradScale : kind == kScaleBf16 ? ldexpf(d, up) : d;
            if (kind >= kScaleCommon && d != 0.f && fabsf(d) <= kMost) {
                int e;
                r = ldexpf(frexpf(d, &e), 15);
                own_alpha = ldexpf(1.f, e - 15);
                ratio = ldexpf(1.f, e - most);
                if (kind == kScaleCommon) r *= ratio;
            }
            if (want < 0 || want >= vocab) r = nan;
        }
        row_scale[i] = r;
        if (kind == kScaleRows) {
            row_alpha[i] = own_alpha;
            row_ratio[i] = ratio;
        }
    }
    if (threadIdx.x == 0) {
        float a = 1.f;
        if (one_finite) {
            a = dloss[0];
            if (mean) a = c > 0 ? a / static_cast<float>(c) : 0.f;
            a /= kLogitGradScale;
        } else if (kind >= kScaleCommon) {
            a = ldexpf(1.f, most - 15);
        } else if (kind == kScaleBf16) {
            a = ldexpf(1.f, -up);
        }
        *alpha = a;
    }
}

// The tiles of a product whose sums came in parts: out = alpha (part 0 + part 1
// + ...) + beta C, added in that order and rounded once. Block (x, y): some rows
// of tile tile0 + y; eight columns per thread. Reads what the parts wrote, mostly
// from L2: a launch more, which the parts have to save (y of one token,
// 2560 x 9728, cold: 42 us whole, 14 + 5 in parts).
struct JoinParams {
    const float* parts;
    int splits, tiles, tile0, tiles_m, tiles_n, group_m, tile_m, tile_n, m, n;
    float alpha, beta;
    const float* alpha_ptr;    // multiplies alpha; may be null
    const float* alpha_rows;   // multiplies alpha, per row; may be null
    const void* c;
    long long ldc;
    void* out;                 // 16-byte aligned rows
    long long ld_out;
    int in_bf16, out_bf16;
};

__global__ void __launch_bounds__(256) join_parts_kernel(const JoinParams p) {
    grid_dependents_launch();
    grid_dependency_wait();
    int tm, tn;
    tile_coords(p.tile0 + static_cast<int>(blockIdx.y), p.tiles_m, p.tiles_n, p.group_m, tm, tn);
    const int per_row = p.tile_n / 8, in_row = static_cast<int>(threadIdx.x) / per_row;
    const int rows = 256 / per_row;                  // of this block; threads beyond have none
    const int r = static_cast<int>(blockIdx.x) * rows + in_row, c = (static_cast<int>(threadIdx.x) - in_row * per_row) * 8;
    const int row = tm * p.tile_m + r, col = tn * p.tile_n + c;
    if (in_row >= rows || r >= p.tile_m || row >= p.m || col >= p.n) return;
    const long long stride = static_cast<long long>(p.tiles) * p.tile_m * p.tile_n;
    const float* src = p.parts + (static_cast<long long>(blockIdx.y) * p.tile_m + r) * p.tile_n + c;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < p.splits; ++k, src += stride) {
        const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
    }
    float alpha = p.alpha_ptr != nullptr ? p.alpha * *p.alpha_ptr : p.alpha;
    if (p.alpha_rows != nullptr) alpha *= p.alpha_rows[row];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= alpha;
    if (p.beta != 0.f) {
        const uint4 w = *(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.c) + row * p.ldc + col));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2(u[i], p.in_bf16);
            v[2 * i] = fmaf(p.beta, f.x, v[2 * i]);
            v[2 * i + 1] = fmaf(p.beta, f.y, v[2 * i + 1]);
        }
    }
    uint4 q;
    q.x = pack2(v[0], v[1], p.out_bf16);
    q.y = pack2(v[2], v[3], p.out_bf16);
    q.z = pack2(v[4], v[5], p.out_bf16);
    q.w = pack2(v[6], v[7], p.out_bf16);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * p.ld_out + col) = q;
}

// ------------------------------------------------------ orthogonalised update ---

// X is kept as FP16 times this power of two: a matrix of Frobenius norm 1 has
// elements near (rows cols)^-1/2, close to FP16's subnormals for large
// matrices; its largest element is at most 1 (and 1.3 after a step), so 256
// leaves room on both sides.
constexpr float kOrthScale = 256.f;

// kOrthScale / norm as two FP32 factors for one after the other, the first a
// power of two (so that the product is rounded once): a single one is infinite
// for norms below 2^-120, which BF16 elements can have.
__device__ __forceinline__ float2 orth_factors(double norm) {
    const double f = static_cast<double>(kOrthScale) / norm;
    // A norm of zero, infinity or NaN gives what the formula gives.
    if (!(f > 0.) || isinf(f)) return make_float2(static_cast<float>(f), 1.f);
    const int half = ilogb(f) / 2;
    return make_float2(static_cast<float>(ldexp(1., half)), static_cast<float>(ldexp(f, -half)));
}

// Eight elements of a row from column c on, zero from `cols` on. kVec: rows are
// 16-byte aligned and whole vectors.
template <bool kVec>
__device__ __forceinline__ void orth_load8(const void* g, long long row, int c, int cols, int bf16, float (&v)[8]) {
    if constexpr (kVec) {
        const uint4 w = *(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(g) + row + c));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = unpack2(u[j], bf16);
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? to_f32(g, row + c + j, bf16) : 0.f;
    }
}

// Elements times `down` have squares within FP32; the result is 1 / down. The
// power of two of the largest of them, or 2^100 from 2^-125 down (whose inverse
// or squares FP32 does not have) and 2^-100 from 2^126 up.
__device__ __forceinline__ double square_scale(float top, float& down) {
    const uint32_t e = __float_as_uint(top) & 0x7f800000u;
    down = e < 0x01000000u ? 0x1p100f : e >= 0x7e800000u ? 0x1p-100f : __uint_as_float(0x7f000000u - e);
    return e < 0x01000000u ? 0x1p-100 : e >= 0x7e800000u ? 0x1p100 : static_cast<double>(__uint_as_float(e));
}

// Sums of squares of matrix blockIdx.y: sums[matrix][block]. Eight squares are
// added in FP32 after dividing by their largest power of two, everything above
// in 64 bits, so that no size of element overflows or is lost. One pass over g
// (16-byte loads, one conversion to 64 bits per eight elements: 9728 x 2560
// takes 19 us cold, element by element in 64 bits it took 114).
template <bool kVec>
__global__ void __launch_bounds__(256) orth_square_kernel(const void* g, long long batch_stride, int rows,
                                                          int cols, long long ld, int bf16,
                                                          double* sums) {
    __shared__ double part[8];
    grid_dependents_launch();
    grid_dependency_wait();
    const long long base = blockIdx.y * batch_stride;
    const int groups = (cols + 7) / 8;
    const long long total = static_cast<long long>(rows) * groups, stride = static_cast<long long>(gridDim.x) * 256;
    double s = 0.;
#pragma unroll 4
    for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total; i += stride) {
        const long long r = i / groups;
        float v[8];
        orth_load8<kVec>(g, base + r * ld, static_cast<int>(i - r * groups) * 8, cols, bf16, v);
        float top = 0.f, sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
        float down;
        const double up = square_scale(top, down);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(v[j] * down, v[j] * down, sum);
        s += static_cast<double>(sum) * up * up;
    }
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) s += part[i];
        sums[static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x] = s;
    }
}

// x = FP16(g kOrthScale / (norm + eps)), rows padded to ld_x (a multiple of 8)
// columns. Memory: 19 us for 9728 x 2560.
template <bool kVec>
__global__ void __launch_bounds__(256) orth_scale_kernel(const void* g, long long batch_stride, int rows,
                                                         int cols, long long ld, int bf16,
                                                         const double* sums, int num_sums, double eps,
                                                         __half* x, long long ld_x, long long x_stride) {
    __shared__ float2 factors;
    grid_dependents_launch();
    grid_dependency_wait();
    if (threadIdx.x < 32) {
        double s = 0.;
        for (int i = threadIdx.x; i < num_sums; i += 32) s += sums[static_cast<long long>(blockIdx.y) * num_sums + i];
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (threadIdx.x == 0) factors = orth_factors(sqrt(s) + eps);
    }
    __syncthreads();
    const float f = factors.x, f2 = factors.y;
    const long long base = blockIdx.y * batch_stride;
    __half* dst = x + blockIdx.y * x_stride;
    const int groups = (cols + 7) / 8;
    const long long total = static_cast<long long>(rows) * groups, stride = static_cast<long long>(gridDim.x) * 256;
#pragma unroll 2
    for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total; i += stride) {
        const long long r = i / groups;
        const int c = static_cast<int>(i - r * groups) * 8;
        float v[8];
        orth_load8<kVec>(g, base + r * ld, c, cols, bf16, v);
        uint4 w;
        w.x = pack2(v[0] * f * f2, v[1] * f * f2, 0);
        w.y = pack2(v[2] * f * f2, v[3] * f * f2, 0);
        w.z = pack2(v[4] * f * f2, v[5] * f * f2, 0);
        w.w = pack2(v[6] * f * f2, v[7] * f * f2, 0);
        *reinterpret_cast<uint4*>(dst + r * ld_x + c) = w;
    }
}

// out[r, c] = scale src[r, c], for outputs whose rows TMA cannot store to (scale
// 1, src in the output's type) and for no step at all (X itself).
__global__ void __launch_bounds__(256) orth_copy_kernel(const void* src, long long ld_src,
                                                        long long src_stride, int src_bf16, float scale,
                                                        void* out, int rows, int cols, int out_bf16) {
    grid_dependents_launch();
    grid_dependency_wait();
    const long long from = blockIdx.y * src_stride, to = static_cast<long long>(blockIdx.y) * rows * cols;
    for (int r = blockIdx.x; r < rows; r += gridDim.x)
        for (int c = threadIdx.x; c < cols; c += 256) {
            const float v = scale * to_f32(src, from + r * ld_src + c, src_bf16);
            const long long i = to + static_cast<long long>(r) * cols + c;
            if (out_bf16) static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
            else static_cast<__half*>(out)[i] = __float2half_rn(v);
        }
}

// All steps of a matrix whose shorter side is at most 128, in one launch: as
// separate launches a step is three kernels of about 4 us each, whose products
// take a tenth of that. A cluster of 1 to 16 CTAs keeps X (shorter side = 128
// rows, zeros below) in shared memory, each CTA `slice` columns of it, in the
// 128-byte-swizzled blocks of 64 columns that serve tcgen05 both as K-major
// operand of X X^T and as MN-major operand of poly X. Per step each CTA
// multiplies its slice's part of X X^T; the parts meet through distributed
// shared memory (CTA r reads rows [128 r / C, 128 (r + 1) / C) of all of them,
// adds them in the order of the CTAs and hands the rounded rows to everyone);
// the polynomial is computed by everyone; X is updated in place. Rounding as in the launches per
// product: FP16 X, X X^T and polynomial, FP32 sums.
// A wait that runs out is recorded and the rest runs on without waiting, since
// all CTAs have to reach the same cluster barriers.
constexpr int kOrthThreads = 256;
constexpr int kOrthMaxSlice = 640;
constexpr uint32_t kOrthBlockBytes = 128u * 128u;                 // 128 rows x 64 halves
constexpr uint32_t kOrthSquareBytes = 2u * kOrthBlockBytes;       // 128 x 128 halves
constexpr uint32_t kOrthMaxSmem = (kOrthMaxSlice / 64) * kOrthBlockBytes + 2 * kOrthSquareBytes + 1024 + 512;
static_assert(kOrthMaxSmem <= 232448, "shared memory");

struct OrthClusterParams {
    const void* g;
    void* out;
    long long batch_stride, ld;
    int side, length;      // shorter and longer side
    int tall;              // the longer side is the rows of g
    int slice;             // columns of X per CTA, a multiple of 64
    int bf16, steps;
    int vec_in, vec_out;   // rows of g / out are 16-byte aligned whole vectors
    float a, b, c;
    double eps;
    int* status;
    unsigned long long timeout_ns;
};

__device__ __forceinline__ void st_dsmem_b64(uint32_t addr, uint32_t lo, uint32_t hi) {
    asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(lo), "r"(hi) : "memory");
}
__device__ __forceinline__ float4 ld_dsmem_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_dsmem_f64(uint32_t addr, double v) {
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

template <uint32_t ctas>
__global__ void __launch_bounds__(kOrthThreads, 1) orth_cluster_kernel(const OrthClusterParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align_1024(smem_raw);
    const uint32_t blocks = static_cast<uint32_t>(p.slice) / 64u;
    uint8_t* xs = smem;                                            // X
    uint8_t* ps = smem + blocks * kOrthBlockBytes;                 // X X^T
    uint8_t* qs = ps + kOrthSquareBytes;                           // polynomial
    float* parts = reinterpret_cast<float*>(ps);                   // [128][128] over both
    uint64_t* bars = reinterpret_cast<uint64_t*>(qs + kOrthSquareBytes);   // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float2* factors = reinterpret_cast<float2*>(tmem_slot + 2);
    double* warp_sums = reinterpret_cast<double*>(bars + 4);       // [8]
    double* cta_sums = warp_sums + 8;                              // [16]

    const uint32_t warp = warp_index(), lane = threadIdx.x & 31u;
    const uint32_t rank = cluster_ctarank();
    auto join_cluster = [&]() {
        __syncwarp();
        cluster_sync();
    };
    const long long base = blockIdx.y * p.batch_stride;
    const int side = p.side, n16 = (side + 15) / 16 * 16;
    const int first = static_cast<int>(rank) * p.slice;
    const int valid = max(0, min(p.slice, p.length - first));      // columns of this slice inside X

    if (threadIdx.x == 0) {
        mbar_init(&bars[0], 1u);
        mbar_init(&bars[1], 1u);
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    for (uint32_t i = threadIdx.x; i < blocks * (kOrthBlockBytes / 16u); i += kOrthThreads)
        reinterpret_cast<uint4*>(xs)[i] = make_uint4(0u, 0u, 0u, 0u);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    grid_dependents_launch();
    grid_dependency_wait();
    const WaitCtl wc{abort_flag, p.status, p.timeout_ns};

    // Where element (s, l) of X lies in shared memory; l counts from this slice.
    auto x_at = [&](int s, int l) {
        return xs + (l >> 6) * kOrthBlockBytes + swz128(static_cast<uint32_t>(s), (l & 63) * 2u);
    };
    // and in g / out, rows `ld` elements apart.
    auto far = [&](long long ld, int s, int l) {
        return p.tall ? (static_cast<long long>(first) + l) * ld + s : s * ld + first + l;
    };
    // Every piece of eight neighbours of a row of g (vector form) or every
    // element, spread over the threads: work(s, l, count). Wide: threads go
    // along the rows. Tall: in the vector form lanes take 32 rows of g, so that
    // their shared-memory accesses are neighbours; else lanes go along a row.
    auto walk = [&](bool vec, auto&& work) {
        if (vec && !p.tall) {
            const int per = valid / 8, n = per * side;
#pragma unroll 4
            for (int q = static_cast<int>(threadIdx.x); q < n; q += kOrthThreads) work(q / per, q % per * 8);
        } else if (vec) {
            const int per = side / 8, n = per * ((valid + 31) / 32);
#pragma unroll 4
            for (int q = static_cast<int>(warp); q < n; q += kOrthThreads / 32) {
                const int l = q / per * 32 + static_cast<int>(lane);
                if (l < valid) work(q % per * 8, l);
            }
        } else {
            const int per = p.tall ? side : valid, n = side * valid;
#pragma unroll 8
            for (int q = static_cast<int>(threadIdx.x); q < n; q += kOrthThreads) {
                const int o = q / per, i = q - o * per;
                work(p.tall ? i : o, p.tall ? o : i);
            }
        }
    };
    // Raw elements into place, and the sum of squares (in 64 bits by pieces, as
    // in orth_square_kernel: no size of element overflows or is lost).
    double sum = 0.;
    if (p.vec_in) {
        walk(true, [&](int s, int l) {
            const uint4 w = *(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.g) + base + far(p.ld, s, l)));
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
            float v[8], top = 0.f, part = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 h = unpack2(u[j >> 1], p.bf16);
                v[j] = (j & 1) ? h.y : h.x;
                top = fmaxf(top, fabsf(v[j]));
                if (p.tall) *reinterpret_cast<uint16_t*>(x_at(s + j, l)) = static_cast<uint16_t>(u[j >> 1] >> ((j & 1) * 16));
            }
            if (!p.tall) *reinterpret_cast<uint4*>(x_at(s, l)) = w;
            float down;
            const double up = square_scale(top, down);
#pragma unroll
            for (int j = 0; j < 8; ++j) part = fmaf(v[j] * down, v[j] * down, part);
            sum += static_cast<double>(part) * up * up;
        });
    } else {
        walk(false, [&](int s, int l) {
            const uint16_t w = *(static_cast<const uint16_t*>(p.g) + base + far(p.ld, s, l));
            *reinterpret_cast<uint16_t*>(x_at(s, l)) = w;
            const double v = static_cast<double>(to_f32(&w, 0, p.bf16));
            sum += v * v;
        });
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sums[warp] = sum;
    __syncthreads();
    if (ctas > 1) join_cluster();   // every CTA of the cluster runs before it is written to
    if (threadIdx.x < ctas) {
        sum = 0.;
        for (int i = 0; i < kOrthThreads / 32; ++i) sum += warp_sums[i];
        st_dsmem_f64(map_to_rank(smem_addr(&cta_sums[rank]), threadIdx.x), sum);
    }
    if (ctas > 1) join_cluster();
    else __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.;
        for (uint32_t i = 0; i < ctas; ++i) sum += cta_sums[i];
        *factors = orth_factors(sqrt(sum) + p.eps);
    }
    __syncthreads();
    const float f = factors->x, f2 = factors->y;
    // Scaled in place (columns outside X are zero).
    for (uint32_t i = threadIdx.x; i < blocks * (kOrthBlockBytes / 16u); i += kOrthThreads) {
        uint4 w = reinterpret_cast<uint4*>(xs)[i];
        uint32_t* u = &w.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 h = unpack2(u[j], p.bf16);
            u[j] = pack2(h.x * f * f2, h.y * f * f2, 0);
        }
        reinterpret_cast<uint4*>(xs)[i] = w;
    }

    const uint32_t x_addr = smem_addr(xs), p_addr = smem_addr(ps), q_addr = smem_addr(qs);
    const uint32_t quarter = warp & 3u, group = warp >> 2;
    const uint32_t row = quarter * 32u + lane;                     // of an accumulator: this thread's
    const bool rows_used = static_cast<int>(quarter * 32u) < side;
    const uint32_t t_row = tmem + ((quarter * 32u) << 16);
    uint32_t phase[2] = {0u, 0u};
    auto wait = [&](int i) {
        mbar_wait(&bars[i], phase[i], wc);
        phase[i] ^= 1u;
        tc_fence_after_sync();
    };
    // Shared-memory writes of all threads before, MMAs after.
    auto hand_over = [&]() {
        fence_async_shared();
        tc_fence_before_sync();
        __syncthreads();
        tc_fence_after_sync();
    };
    // 32 columns from `col` of this thread's row in swizzled blocks, as FP16 (or BF16).
    auto put_square = [&](uint8_t* dst, uint32_t col, const float (&v)[32], int bf16 = 0) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            uint4 w;
            w.x = pack2(v[8 * j], v[8 * j + 1], bf16);
            w.y = pack2(v[8 * j + 2], v[8 * j + 3], bf16);
            w.z = pack2(v[8 * j + 4], v[8 * j + 5], bf16);
            w.w = pack2(v[8 * j + 6], v[8 * j + 7], bf16);
            *reinterpret_cast<uint4*>(dst + (col >> 6) * kOrthBlockBytes + swz128(row, (col & 63u) * 2u + 16u * j)) = w;
        }
    };
    auto get_row = [&](const uint8_t* src, uint32_t col, float (&v)[32]) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint4 w = *reinterpret_cast<const uint4*>(src + (col >> 6) * kOrthBlockBytes +
                                                            swz128(row, (col & 63u) * 2u + 16u * j));
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 h = unpack2(u[i], 0);
                v[8 * j + 2 * i] = h.x;
                v[8 * j + 2 * i + 1] = h.y;
            }
        }
    };
    const uint32_t square_idesc = make_idesc_f16(128, 0, false, false) | (static_cast<uint32_t>(n16 >> 3) << 17);
    const float inv = 1.f / kOrthScale;
    constexpr uint32_t own = 128u / ctas;                          // rows of X X^T that this CTA sums

    for (int step = 0; step < p.steps; ++step) {
        const bool last = step + 1 == p.steps;
        // X X^T of this slice.
        hand_over();
        if (warp == 0) {
            const uint32_t issuer = elect_lane();
            uint32_t add = 0;
            for (uint32_t j = 0; j < blocks; ++j) {
                const uint64_t d = make_smem_desc(x_addr + j * kOrthBlockBytes, 16u, 1024u);
#pragma unroll
                for (uint32_t kk = 0; kk < 4; ++kk) {
                    tc_mma_if<false>(issuer, tmem, d + kk * 2u, d + kk * 2u, square_idesc, add);
                    add = 1;
                }
            }
            tc_commit_if<false>(issuer, smem_addr(&bars[0]));
        }
        wait(0);
        if constexpr (ctas == 1) {
            for (uint32_t c = 32u * group; rows_used && static_cast<int>(c) < n16; c += 64u) {
                float v[32];
                tmem_ld32(t_row + c, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] *= inv * inv;
                put_square(ps, c, v);
            }
        } else {
            // This slice's part over both squares, which no MMA reads now; a
            // row's 16-byte pieces are permuted by its number, so that lanes
            // (rows) write to different banks.
            for (uint32_t c = 32u * group; rows_used && static_cast<int>(c) < n16; c += 64u) {
                float v[32];
                tmem_ld32(t_row + c, v);
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    reinterpret_cast<float4*>(parts)[row * 32u + ((c / 4u + i) ^ (row & 7u))] =
                        make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
            tc_fence_before_sync();
            join_cluster();
            // This CTA's rows of all the parts: 16 pieces of four columns a thread
            // whatever the cluster's size, all in flight, then added in order.
            constexpr uint32_t kTurns = 16 / ctas;
            float4 w[16];
#pragma unroll
            for (uint32_t k = 0; k < kTurns; ++k) {
                const uint32_t q = k * kOrthThreads + threadIdx.x, r = rank * own + q / 32u, piece = q & 31u;
                const uint32_t at = smem_addr(parts) + (r * 32u + (piece ^ (r & 7u))) * 16u;
                const bool wanted = static_cast<int>(r) < n16 && static_cast<int>(piece * 4u) < n16;
#pragma unroll
                for (uint32_t from = 0; from < ctas; ++from)
                    w[k * ctas + from] = wanted ? ld_dsmem_f4(map_to_rank(at, from)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            uint32_t sums[kTurns][2];
#pragma unroll
            for (uint32_t k = 0; k < kTurns; ++k) {
                float4 a = w[k * ctas];
#pragma unroll
                for (uint32_t from = 1; from < ctas; ++from) {
                    const float4 u = w[k * ctas + from];
                    a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
                }
                sums[k][0] = pack2(a.x * inv * inv, a.y * inv * inv, 0);
                sums[k][1] = pack2(a.z * inv * inv, a.w * inv * inv, 0);
            }
            join_cluster();
#pragma unroll
            for (uint32_t k = 0; k < kTurns; ++k) {
                const uint32_t q = k * kOrthThreads + threadIdx.x;
                const uint32_t r = rank * own + q / 32u, col = (q & 31u) * 4u;
                if (static_cast<int>(r) < n16 && static_cast<int>(col) < n16) {
                    const uint32_t at = p_addr + (col >> 6) * kOrthBlockBytes + swz128(r, (col & 63u) * 2u);
#pragma unroll
                    for (uint32_t to = 0; to < ctas; ++to) st_dsmem_b64(map_to_rank(at, to), sums[k][0], sums[k][1]);
                }
            }
            // The rows come from other CTAs: each side orders them towards the MMAs.
            fence_async_shared();
            join_cluster();
        }
        // b P + c P P
        hand_over();
        if (warp == 0) {
            const uint32_t issuer = elect_lane();
            for (int k = 0; k < n16; k += 16) {
                const uint64_t d = make_smem_desc(p_addr + (k >> 6) * kOrthBlockBytes, 16u, 1024u) + ((k & 63) >> 3);
                tc_mma_if<false>(issuer, tmem + 256u, d, d, square_idesc, k > 0 ? 1u : 0u);
            }
            tc_commit_if<false>(issuer, smem_addr(&bars[0]));
        }
        wait(0);
        for (uint32_t c = 32u * group; rows_used && static_cast<int>(c) < n16; c += 64u) {
            float v[32], w[32];
            tmem_ld32(t_row + 256u + c, v);
            get_row(ps, c, w);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = fmaf(p.c, v[i], p.b * w[i]);
            put_square(qs, c, v);
        }
        // X <- a X + poly X, 256 columns at a time, two accumulators in turn.
        hand_over();
        const int turns = (p.slice + 255) / 256;
        auto update = [&](int turn) {
            if (warp != 0) return;
            const uint32_t issuer = elect_lane();
            const int width = min(256, p.slice - 256 * turn);
            const uint32_t idesc = make_idesc_f16(128, 0, false, true) | (static_cast<uint32_t>(width >> 3) << 17);
            const uint64_t db = make_smem_desc(x_addr + turn * 4 * kOrthBlockBytes, kOrthBlockBytes, 1024u);
            for (int k = 0; k < n16; k += 16) {
                const uint64_t da = make_smem_desc(q_addr + (k >> 6) * kOrthBlockBytes, 16u, 1024u) + ((k & 63) >> 3);
                tc_mma_if<false>(issuer, tmem + (turn & 1) * 256u, da, db + static_cast<uint64_t>(k) * 8u, idesc,
                                 k > 0 ? 1u : 0u);
            }
            tc_commit_if<false>(issuer, smem_addr(&bars[turn & 1]));
        };
        update(0);
        if (turns > 1) update(1);
        for (int turn = 0; turn < turns; ++turn) {
            wait(turn & 1);
            const uint32_t width = static_cast<uint32_t>(min(256, p.slice - 256 * turn));
            for (uint32_t c = 32u * group; rows_used && c < width; c += 64u) {
                const uint32_t col = 256u * turn + c;
                if (static_cast<int>(col) >= valid) break;
                float v[32], w[32];
                tmem_ld32(t_row + (turn & 1) * 256u + c, v);
                get_row(xs, col, w);
                const float a = last ? p.a * inv : p.a, scale = last ? inv : 1.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = fmaf(scale, v[i], a * w[i]);
                if (static_cast<int>(row) < side) put_square(xs, col, v, last ? p.bf16 : 0);
                __syncwarp();
            }
            if (turn + 2 < turns) {
                tc_fence_before_sync();
                __syncthreads();
                tc_fence_after_sync();
                update(turn + 2);
            }
        }
        // A CTA's squares are next written by itself, and by others only once it
        // has come to the next step's second barrier.
    }
    tc_fence_before_sync();
    __syncthreads();
    // X, now in the type of the result, to memory.
    uint16_t* out = static_cast<uint16_t*>(p.out) + static_cast<long long>(blockIdx.y) * side * p.length;
    const long long ld_out = p.tall ? side : p.length;
    if (p.vec_out) {
        walk(true, [&](int s, int l) {
            uint4 w;
            if (!p.tall) {
                w = *reinterpret_cast<const uint4*>(x_at(s, l));
            } else {
                uint32_t u[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] = *reinterpret_cast<const uint16_t*>(x_at(s + j, l));
                w = make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
            }
            *reinterpret_cast<uint4*>(out + far(ld_out, s, l)) = w;
        });
    } else {
        walk(false, [&](int s, int l) { out[far(ld_out, s, l)] = *reinterpret_cast<const uint16_t*>(x_at(s, l)); });
    }
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
    if (ctas > 1) join_cluster();   // no CTA leaves while others may read its part
}

}  // namespace hgemm
