// Product of two 8-bit matrices with scales for blocks of 128 on the tensor
// cores, and its C entry points (include/mdsoap.h).
//
//   out[i][j] = sum_b sa[i][b] sb[j'][b] (sum over k in block b of a[i][k] b[j][k])
//
// The inner sums are matrix instructions over 128 bytes of K into tensor memory.
// Their scales change from block to block, so each block's partial product is
// taken out of tensor memory, multiplied and added in float32 registers, while
// the next block fills the other accumulator.
#include "readout_host.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <type_traits>

using namespace mdsoap;
using namespace mdsoap::readout;

namespace {

constexpr int kTileK = 128;  // bytes of K a stage: one scale block
constexpr int kRows = 128;   // rows of one CTA's accumulator: the lanes of tensor memory

__device__ unsigned g_gave_up;  // products whose copies or matrix instructions did not complete in time

struct ProductArgs {
    int64_t m, n, k;
    const float* a_scales;
    int64_t a_scale_stride;
    const float* b_scales;
    int64_t b_scale_stride;
    int32_t b_tiles;
    void* out;
    int64_t out_stride;
    int32_t accumulate;
    int32_t splits;   // parts of K, each a work item of its own
    float* partials;  // [split][tile][256][256] where splits > 1
    int32_t copies[2];  // blocks that the first and the second CTA of a pair copy at most; negative: all (mdsoap_probe_matmul)
};

// Four neighbouring scales of a row from block `b` on; zero from block `end` on.
__device__ __forceinline__ float4 scales4(const float* row, int b, int end, bool vector) {
    if (vector && b + 4 <= end) return __ldg(reinterpret_cast<const float4*>(row + b));
    float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (b < end) f.x = row[b];
    if (b + 1 < end) f.y = row[b + 1];
    if (b + 2 < end) f.z = row[b + 2];
    if (b + 3 < end) f.w = row[b + 3];
    return f;
}

__device__ __forceinline__ float pick(const float4& f, int i) {
    const float low = i & 1 ? f.y : f.x, high = i & 1 ? f.w : f.z;
    return i & 2 ? high : low;
}

// COUNT neighbouring results of one row; `left` of them lie inside the matrix.
template <class OUT, int COUNT>
__device__ __forceinline__ void store_row(OUT* p, int64_t left, const float (&f)[COUNT], bool add) {
#pragma unroll
    for (int i = 0; i < COUNT; i += 4) {
        float v[4] = {f[i], f[i + 1], f[i + 2], f[i + 3]};
        if (i + 4 <= left && reinterpret_cast<uintptr_t>(p + i) % (4 * sizeof(OUT)) == 0) {
            if constexpr (sizeof(OUT) == 4) {
                float4* q = reinterpret_cast<float4*>(p + i);
                if (add) {
                    const float4 o = *q;
                    v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
                }
                *q = make_float4(v[0], v[1], v[2], v[3]);
            } else {
                uint2 q;
                OUT* t = reinterpret_cast<OUT*>(&q);
#pragma unroll
                for (int j = 0; j < 4; ++j) t[j] = from_float<OUT>(v[j]);
                *reinterpret_cast<uint2*>(p + i) = q;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < left) p[i + j] = from_float<OUT>(add ? to_float(p[i + j]) + v[j] : v[j]);
        }
    }
}

// ------------------------------------------------------------ pairs of CTAs
//
// A pair of CTAs (two SMs) computes a tile of 256 x 256: each holds 128 rows of
// A and of B in shared memory and 128 rows of the accumulators, and the pair's
// matrix instructions read both halves of B, so each SM copies and reads only
// half of it.  A single SM's 128 x 256 tile would move 48 KB through shared
// memory for every 128 of K where this moves 32 KB; at the tensor cores' rate
// that is what shared memory can deliver.
// Per CTA: warp 8 copies tiles of A and B (one block of K a stage), warp 9 of
// the first CTA issues the matrix instructions, warps 0 to 7 scale and add.
// Persistent: the pairs take tiles (and parts of K) in turn, columns first, so
// that the pairs at work share A's rows and B stays in L2.
//
// Measured: 131 072 x 4096 x 3696 into bfloat16 2.41 to 2.48 ms, 1.6 PFLOP/s, with
// the board at its power limit (1.65 GHz at 1000 W); 128 x 128 tiles of one CTA
// took 3.95 ms.  Two accumulators fill tensor memory, so a block's matrix
// instructions (512 clocks) wait until its accumulator of two blocks ago has been
// read: commit, wake, read and arrival take another 1000 to 1500 clocks for every
// two blocks.  Without the multiplications the same loop takes 2.0 ms, without
// reading tensor memory 1.9, the copies alone 1.4 (10.8 TB/s out of L2).  Four
// accumulators of half the columns took 2.7 ms (each instruction reads A again),
// sixteen warps with half the columns each 2.8 (registers).
// Scales of B's rows instead of tiles cost a multiplication and a read of shared
// memory more for every product: 1024 x 2100 x 65 537 into float32 280 us, 1.0
// PFLOP/s.

constexpr int kPairTile = 256;
constexpr int kPromote = 8;                    // warps that scale and add the partial products
constexpr int kMine = kPairTile / (kPromote / 4);  // columns of one of their threads
constexpr int kThreads = (kPromote + 4) * 32;  // a warp each for the copies and the matrix instructions, two to fill up
// Registers: launched with 168 a thread; the last four warps give theirs up to 72
// and the other eight take 216 (8 x 216 + 4 x 72 = 12 x 168).
constexpr int kManyRegisters = 216, kFewRegisters = 72;

enum class Store { Tile, Direct, Partial };

template <bool TILES>
struct PairShared {
    static constexpr int kStages = 5;
    static constexpr int kOut = TILES ? 2 : 1;  // pieces of a warp's results on their way out at a time
    uint8_t a[kStages][kRows * kTileK];
    uint8_t b[kStages][kRows * kTileK];
    uint8_t out[kOut][kPromote][32 * 128];  // 128-byte pieces of a warp's 32 rows
    float b_scale[TILES ? 1 : 2][4][TILES ? 4 : kPairTile];
    uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], drained;
    uint32_t tensor_memory;
    int gave_up, other_gave_up;  // this CTA, the pair's other one
    int issued;
};

constexpr int kStep = 16;  // columns that leave tensor memory at a time

// acc + part x scale for a pair of columns.  Two scalar fmas: as one packed
// fma.f32x2 the pairs needed as many register moves as it saved instructions.
__device__ __forceinline__ uint64_t add_scaled(uint32_t x, uint32_t y, uint64_t scale, uint64_t acc) {
    float m0, m1, a0, a1;
    tc::split_pair(scale, m0, m1);
    tc::split_pair(acc, a0, a1);
    return tc::pair_of(fmaf(__uint_as_float(x), m0, a0), fmaf(__uint_as_float(y), m1, a1));
}

// A warp's piece of 32 rows x 128 bytes from (swizzled) shared memory to rows of
// a matrix, BYTES at a time; `rows` rows and `cols` elements of each exist.
// WHOLE: all of them, and nothing is added, so that reads and writes need not wait
// for one another.
template <class OUT, int BYTES, bool WHOLE>
__device__ __forceinline__ void copy_rows(const uint8_t* from, OUT* out, int64_t stride, int rows, int cols, bool add) {
    using Word = std::conditional_t<BYTES == 8, uint2, std::conditional_t<BYTES == 4, uint32_t, uint16_t>>;
    constexpr int kAcross = 128 / BYTES;                       // words of a row
    constexpr int kLanes = kAcross < 32 ? kAcross : 32;        // lanes on one row
    constexpr int kRowsAtOnce = 32 / kLanes;
    const int lane = threadIdx.x & 31;
    out += lane / kLanes * stride + lane % kLanes * (BYTES / (int)sizeof(OUT));
#pragma unroll 8
    for (int i = 0; i < kLanes; ++i, out += kRowsAtOnce * stride) {
        const int r = i * kRowsAtOnce + lane / kLanes;
        if (!WHOLE && r >= rows) break;
#pragma unroll
        for (int k = 0; k < kAcross / kLanes; ++k) {
            const int byte = (k * kLanes + lane % kLanes) * BYTES;
            const Word w = *reinterpret_cast<const Word*>(from + r * 128 + ((byte / 16 ^ (r & 7)) * 16) + byte % 16);
            Word* to = reinterpret_cast<Word*>(out + k * kLanes * (BYTES / (int)sizeof(OUT)));
            if constexpr (WHOLE) {
                *to = w;
            } else {
                if (byte / (int)sizeof(OUT) >= cols) continue;
                if (add) {
                    Word sum = *to;
                    OUT* t = reinterpret_cast<OUT*>(&sum);
                    const OUT* v = reinterpret_cast<const OUT*>(&w);
#pragma unroll
                    for (int j = 0; j < BYTES / (int)sizeof(OUT); ++j) t[j] = from_float<OUT>(to_float(t[j]) + to_float(v[j]));
                    *to = sum;
                } else {
                    *to = w;
                }
            }
        }
    }
}

template <class OUT, int BYTES>
__device__ __forceinline__ void copy_rows(const uint8_t* from, OUT* out, int64_t stride, int rows, int cols, bool add) {
    if (rows >= 32 && cols >= 128 / (int)sizeof(OUT) && !add) copy_rows<OUT, BYTES, true>(from, out, stride, rows, cols, false);
    else copy_rows<OUT, BYTES, false>(from, out, stride, rows, cols, add);
}

// NaN into a warp's 32 rows x kMine columns, of which `rows` and `cols` exist.
template <class OUT>
__device__ __forceinline__ void fill_nan(OUT* out, int64_t stride, int64_t rows, int64_t cols) {
#pragma unroll 1
    for (int i = 0; i < 32 && i < rows; ++i, out += stride)
#pragma unroll 1
        for (int c = threadIdx.x & 31; c < kMine && c < cols; c += 32) out[c] = from_float<OUT>(__int_as_float(-1));
}

template <bool TILES, class OUT, Store STORE>
__global__ __launch_bounds__(kThreads, 1) void pair_product_kernel(const __grid_constant__ CUtensorMap map_a,
                                                                   const __grid_constant__ CUtensorMap map_b,
                                                                   const __grid_constant__ CUtensorMap map_out,
                                                                   const __grid_constant__ ProductArgs p) {
    extern __shared__ uint8_t raw[];
    using S = PairShared<TILES>;
    constexpr int kStages = S::kStages;
    S& s = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)tc::cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int blocks = (int)((p.k + kTileK - 1) / kTileK);
    const int tiles_n = (int)((p.n + kPairTile - 1) / kPairTile), tiles_m = (int)((p.m + kPairTile - 1) / kPairTile);
    const int tiles = tiles_n * tiles_m, items = tiles * p.splits;  // the host keeps them below 2^30

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            bulk::barrier_init(&s.full[i], 1);
            bulk::barrier_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            bulk::barrier_init(&s.acc_full[i], 1);
            bulk::barrier_init(&s.acc_empty[i], 2 * kPromote);  // both CTAs' warps
        }
        bulk::barrier_init(&s.drained, 1);
        s.gave_up = s.other_gave_up = 0;
        s.issued = 0;
        bulk::barrier_init_fence();
    }
    if (threadIdx.x == kPromote * 32) {
        tc::prefetch_map(&map_a);
        tc::prefetch_map(&map_b);
    }
    if (warp == kPromote + 1) tc::alloc<2>(&s.tensor_memory, 512);
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();
    tc::fence_after();
    const uint32_t tmem = *(volatile uint32_t*)&s.tensor_memory;
    volatile int* gave_up = &s.gave_up;

    // The tile and the part of K of a work item.
    const auto item_m = [&](int item) { return item % tiles / tiles_n * kPairTile; };
    const auto item_n = [&](int item) { return item % tiles % tiles_n * kPairTile; };
    const auto first_block = [&](int item) { return (int)((int64_t)(item / tiles) * blocks / p.splits); };
    const auto last_block = [&](int item) { return (int)((int64_t)(item / tiles + 1) * blocks / p.splits); };

    if (warp >= kPromote) {
        tc::give_registers<kFewRegisters>();
        if (warp == kPromote && lane == 0) {
            const int most = p.copies[rank];
            int stage = 0, phase = 0, count = 0;
            bool good = true;
            for (int item = pair; item < items && good; item += pairs) {
                const int m0 = item_m(item) + rank * kRows, n0 = item_n(item) + rank * kRows;
                const int end = last_block(item);
                for (int kb = first_block(item); kb < end; ++kb, ++count) {
                    if (count == most || !tc::wait(&s.empty[stage], phase ^ 1, gave_up)) {
                        good = false;
                        break;
                    }
                    const uint32_t full = tc::map_shared(&s.full[stage], 0);
                    if (rank == 0) bulk::arrive_expect(&s.full[stage], 4 * kRows * kTileK);
                    tc::load_tile_pair(s.a[stage], &map_a, kb * kTileK, m0, full);
                    tc::load_tile_pair(s.b[stage], &map_b, kb * kTileK, n0, full);
                    if (++stage == kStages) stage = 0, phase ^= 1;
                }
            }
            s.issued = count;
        } else if (warp == kPromote + 1 && lane == 0 && rank == 0) {
            constexpr uint32_t word = tc::instruction(kPairTile, kPairTile);
            constexpr int kStep16 = kRows * kTileK / 16;  // descriptors count in units of 16 bytes
            const uint64_t first_a = tc::operand(s.a[0]), first_b = tc::operand(s.b[0]);
            int stage = 0, phase = 0, parity = 0, turn = 0;
            bool good = true;
            for (int item = pair; item < items && good; item += pairs) {
                for (int left = last_block(item) - first_block(item); left > 0; --left) {
                    const uint64_t a = first_a + stage * kStep16, b = first_b + stage * kStep16;
                    const uint32_t d = tmem + parity * kPairTile;
                    good = tc::wait(&s.full[stage], phase, gave_up) && tc::wait(&s.acc_empty[parity], turn ^ 1, gave_up);
                    if (!good) break;
                    tc::fence_after();
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc::mma<2>(d, a + 2 * k, b + 2 * k, word, k > 0);
                    tc::commit<2>(&s.acc_full[parity]);
                    tc::commit<2>(&s.empty[stage]);
                    if (++stage == kStages) stage = 0, phase ^= 1;
                    parity ^= 1;
                    turn ^= parity ^ 1;  // after every second block
                }
            }
            if (!good) {  // matrix instructions in flight end before the tensor memory goes
                tc::commit<2>(&s.drained);
                bulk::wait(&s.drained, 0);
            }
        }
    } else {
        tc::take_registers<kManyRegisters>();
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + half * kMine;
        const uint32_t empty0 = tc::map_shared(&s.acc_empty[0], 0);
        const bool vec_a = p.a_scale_stride % 4 == 0 && reinterpret_cast<uintptr_t>(p.a_scales) % 16 == 0;
        const bool vec_b = p.b_scale_stride % 4 == 0 && reinterpret_cast<uintptr_t>(p.b_scales) % 16 == 0;
        int parity = 0, turn = 0;
        // The half of b_scale that a turn fills.  It alternates through the whole kernel, from one item to the next
        // too: the barrier of the turn between lets nobody fill a half that a slower warp still reads.
        int group = 0, item = pair;
        for (; item < items; item += pairs) {
            const int m0 = item_m(item) + rank * kRows, n0 = item_n(item);
            const int begin = first_block(item), end = last_block(item);
            const int row = m0 + quarter * 32 + lane, col = n0 + half * kMine;
            // a row or column past the matrix takes scales of one that exists; its results are never stored
            const float* sa = p.a_scales + min(row, (int)p.m - 1) * p.a_scale_stride;
            const float* sb = p.b_scales +
                              (TILES ? min(col, (int)p.n - 1) / kBlock : min(n0 + (int)threadIdx.x, (int)p.n - 1)) *
                                  p.b_scale_stride;
            uint64_t acc[kMine / 2];
#pragma unroll
            for (int i = 0; i < kMine / 2; ++i) acc[i] = 0;  // two zeros
            float4 next_a = scales4(sa, begin & ~3, end, vec_a), next_b = scales4(sb, begin & ~3, end, vec_b);
            // four blocks a turn: their scales were loaded one turn ahead
            for (int first = begin & ~3; first < end; first += 4) {
                float scale[4] = {next_a.x, next_a.y, next_a.z, next_a.w};
                group ^= 1;
                if constexpr (TILES) {
                    scale[0] *= next_b.x, scale[1] *= next_b.y, scale[2] *= next_b.z, scale[3] *= next_b.w;
                } else {
                    s.b_scale[group][0][threadIdx.x] = next_b.x;
                    s.b_scale[group][1][threadIdx.x] = next_b.y;
                    s.b_scale[group][2][threadIdx.x] = next_b.z;
                    s.b_scale[group][3][threadIdx.x] = next_b.w;
                    // the four warps that share a half of the columns
                    asm volatile("bar.sync %0, %1;" ::"r"(1 + half), "n"(kRows) : "memory");
                }
                next_a = scales4(sa, first + 4, end, vec_a);
                next_b = scales4(sb, first + 4, end, vec_b);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (first + j < begin || first + j >= end) continue;
                    const uint64_t mine2 = tc::pair_of(scale[j], scale[j]);
                    const uint32_t from = lanes + parity * kPairTile;
                    const ulonglong2* sb2 =
                        reinterpret_cast<const ulonglong2*>(&s.b_scale[TILES ? 0 : group][j][TILES ? 0 : half * kMine]);
                    tc::wait(&s.acc_full[parity], turn, gave_up);
                    __syncwarp();
                    tc::fence_after();
                    // the next columns leave tensor memory while these are added
                    uint32_t part[2][kStep];
                    tc::load(from, part[0]);
#pragma unroll
                    for (int c = 0; c < kMine; c += kStep) {
                        tc::wait_loads();
                        if (c + kStep < kMine) {
                            tc::load(from + c + kStep, part[(c / kStep + 1) & 1]);
                        } else {
                            tc::fence_before();
                            __syncwarp();
                            if (lane == 0) tc::arrive_at(empty0 + parity * (uint32_t)sizeof(uint64_t));
                        }
                        const uint32_t(&now)[kStep] = part[c / kStep & 1];
                        if constexpr (TILES) {
#pragma unroll
                            for (int i = 0; i < kStep / 2; ++i)
                                acc[c / 2 + i] = add_scaled(now[2 * i], now[2 * i + 1], mine2, acc[c / 2 + i]);
                        } else {
#pragma unroll
                            for (int i = 0; i < kStep / 2; i += 2) {
                                const ulonglong2 q = sb2[(c + 2 * i) / 4];
                                acc[c / 2 + i] = add_scaled(now[2 * i], now[2 * i + 1], tc::mul2(mine2, q.x), acc[c / 2 + i]);
                                acc[c / 2 + i + 1] =
                                    add_scaled(now[2 * i + 2], now[2 * i + 3], tc::mul2(mine2, q.y), acc[c / 2 + i + 1]);
                            }
                        }
                    }
                    parity ^= 1;
                    turn ^= parity ^ 1;
                }
            }
            if (tc::any_of(1 + half, kRows, *gave_up)) break;  // together: a half's warps meet at barriers
            if constexpr (STORE == Store::Partial && !TILES) {
                // straight out of the registers: through the copy engine, as below, a part of few blocks ends 4 us
                // earlier, but this form's loop, short of registers, loses more (1024 x 2100 x 65 537: 281 -> 329 us)
                float* out = p.partials + ((int64_t)item * kPairTile + rank * kRows + quarter * 32 + lane) * kPairTile + half * kMine;
#pragma unroll
                for (int i = 0; i < kMine / 2; i += 2)
                    *reinterpret_cast<ulonglong2*>(out + 2 * i) = make_ulonglong2(acc[i], acc[i + 1]);
            } else {
                // 128 bytes of each of the warp's rows at a time, through shared memory: 16-byte pieces in the
                // swizzled order the copy engine expects (piece ^ row % 8), so that no side meets bank conflicts
                constexpr int kWide = 128 / (int)sizeof(OUT), kEach = 16 / (int)sizeof(OUT);
                const int row0 = m0 + quarter * 32;
#pragma unroll
                for (int c = 0; c < kMine; c += kWide) {
                    uint8_t* const piece_out = s.out[c / kWide % S::kOut][warp];
                    uint8_t* const piece_row = piece_out + lane * 128;
                    if (STORE != Store::Direct && lane == 0) tc::wait_store_reads<S::kOut - 1>();
                    __syncwarp();
#pragma unroll
                    for (int piece = 0; piece < 8; ++piece) {
                        float f[kEach];
#pragma unroll
                        for (int i = 0; i < kEach; i += 2)
                            tc::split_pair(acc[(c + piece * kEach + i) / 2], f[i], f[i + 1]);
                        uint4 q;
                        if constexpr (sizeof(OUT) == 4)
                            q = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                           __float_as_uint(f[3]));
                        else
                            q = make_uint4(pack2<OUT>(f[0], f[1]), pack2<OUT>(f[2], f[3]), pack2<OUT>(f[4 % kEach], f[5 % kEach]),
                                           pack2<OUT>(f[6 % kEach], f[7 % kEach]));
                        *reinterpret_cast<uint4*>(piece_row + ((piece ^ (lane & 7)) * 16)) = q;
                    }
                    if constexpr (STORE == Store::Tile) {
                        bulk::proxy_fence();
                        __syncwarp();
                        if (lane == 0) {
                            if (row0 < p.m && col + c < p.n) tc::store_tile(&map_out, col + c, row0, piece_out);
                            tc::end_stores();  // a group a piece, so that the wait counts pieces
                        }
                    } else if constexpr (STORE == Store::Partial) {
                        bulk::proxy_fence();
                        __syncwarp();
                        if (lane == 0) {
                            tc::store_tile(&map_out, half * kMine + c, item * kPairTile + rank * kRows + quarter * 32,
                                           piece_out);
                            tc::end_stores();
                        }
                    } else {
                        // rows that the copy engine cannot write, or that are added to: words as wide as the
                        // rows' alignment allows, neighbouring lanes on neighbouring words
                        __syncwarp();
                        OUT* const out = static_cast<OUT*>(p.out) + (int64_t)row0 * p.out_stride + col + c;
                        const int rows = min(32, (int)p.m - row0), cols = (int)p.n - col - c;
                        const uintptr_t mixed = reinterpret_cast<uintptr_t>(out) |
                                                (uintptr_t)(p.out_stride * (int64_t)sizeof(OUT)) |
                                                (uintptr_t)(min(cols, kWide) * (int)sizeof(OUT));
                        if (cols <= 0) continue;
                        if (mixed % 8 == 0) copy_rows<OUT, 8>(piece_out, out, p.out_stride, rows, cols, p.accumulate);
                        else if (mixed % 4 == 0) copy_rows<OUT, 4>(piece_out, out, p.out_stride, rows, cols, p.accumulate);
                        else copy_rows<OUT, sizeof(OUT)>(piece_out, out, p.out_stride, rows, cols, p.accumulate);
                    }
                }
            }
        }
        // what a half that gave up owes becomes NaN
#pragma unroll 1
        for (; item < items; item += pairs) {
            const int64_t row0 = item_m(item) + rank * kRows + quarter * 32, col0 = item_n(item) + half * kMine;
            if constexpr (STORE == Store::Partial)
                fill_nan(p.partials + ((int64_t)item * kPairTile + rank * kRows + quarter * 32) * kPairTile + half * kMine,
                         kPairTile, 32, kMine);
            else
                fill_nan(static_cast<OUT*>(p.out) + row0 * p.out_stride + col0, p.out_stride, p.m - row0, p.n - col0);
        }
        if (STORE != Store::Direct && lane == 0) tc::wait_store_reads<0>();  // before the shared memory goes
    }

    __syncthreads();
    if (*gave_up && threadIdx.x == 0) {
        atomicOr(&g_gave_up, 1u);
        tc::store_shared_at(tc::map_shared(&s.other_gave_up, rank ^ 1), 1);
    }
    tc::cluster_sync();  // neither CTA leaves while the other may still reach into its memory
    if (*gave_up || *(volatile int*)&s.other_gave_up) {
        // Both CTAs' copies in flight land before their shared memory goes.  The first CTA's barriers count them, and
        // it announced both CTAs' bytes for the blocks that it copied; one of the two may have stopped earlier.
        if (rank == 0 && threadIdx.x == 0) {
            constexpr uint32_t kEach = 2 * kRows * kTileK;  // bytes of a block that one CTA copies
            const int mine = s.issued, other = tc::load_int_at(tc::map_shared(&s.issued, 1)), all = max(mine, other);
            for (int i = min(mine, other); i < all; ++i) {
                if (mine < other) bulk::arrive_expect(&s.full[i % kStages], kEach);
                else tc::complete_bytes(&s.full[i % kStages], kEach);
            }
            for (int i = max(0, all - kStages); i < all; ++i) bulk::wait(&s.full[i % kStages], i / kStages & 1);
        }
        tc::cluster_sync();
    }
    if (warp == kPromote + 1) tc::dealloc<2>(tmem, 512);
}

// out = the parts' partial products in order.
template <class OUT>
__global__ __launch_bounds__(256) void add_parts_kernel(const __grid_constant__ ProductArgs p) {
    const int tiles_n = (int)((p.n + kPairTile - 1) / kPairTile), tiles_m = (int)((p.m + kPairTile - 1) / kPairTile);
    const int64_t part = (int64_t)tiles_n * tiles_m * kPairTile * kPairTile;
    const int64_t col = (blockIdx.x * 64ll + threadIdx.x % 64) * 4;
    if (col >= p.n) return;
    for (int64_t row = blockIdx.y * 4ll + threadIdx.x / 64; row < p.m; row += gridDim.y * 4ll) {
        const float* from = p.partials + ((row / kPairTile * tiles_n + col / kPairTile) * kPairTile + row % kPairTile) * kPairTile +
                            col % kPairTile;
        float4 sum = *reinterpret_cast<const float4*>(from);
#pragma unroll 4
        for (int i = 1; i < p.splits; ++i) {
            const float4 q = *reinterpret_cast<const float4*>(from + i * part);
            sum.x += q.x, sum.y += q.y, sum.z += q.z, sum.w += q.w;
        }
        const float f[4] = {sum.x, sum.y, sum.z, sum.w};
        store_row(static_cast<OUT*>(p.out) + row * p.out_stride + col, p.n - col, f, p.accumulate);
    }
}

// ------------------------------------------------------------ few rows
//
// With at most 128 rows of A the product reads B once and is bound by that.
// Here B's rows are the lanes: a CTA takes 128 of them and all rows of A (padded
// to COLS) as the columns, so each 16 KB of B travel beside COLS / 8 KB of A.
// The CTAs of a cluster share K, each adds up its part, and they join their sums
// through each other's shared memory in the cluster's order.
// One row x 1024 x 3696: 6.4 us back to back on the device (9.3 us a call from
// Python), of which its 3.8 MB take 0.6 us: launch, cluster barriers and the first
// copies' latency are the rest.

constexpr int kFewThreads = 6 * 32;  // four warps that scale and add, one for the copies, one for the instructions

template <int COLS>
struct FewShared {  // at most 224 KB
    static constexpr int kStages = COLS <= 32 ? 8 : COLS == 64 ? 7 : 4;
    uint8_t b[kStages][kRows * kTileK];
    uint8_t a[kStages][COLS * kTileK];
    float a_scale[2][4][COLS];
    float sum[COLS][kRows];
    uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], drained;
    uint32_t tensor_memory;
    int gave_up;
    int issued;
};

template <int COLS, class OUT>
__global__ __launch_bounds__(kFewThreads, 1) void few_product_kernel(const __grid_constant__ CUtensorMap map_a,
                                                                     const __grid_constant__ CUtensorMap map_b,
                                                                     const __grid_constant__ ProductArgs p) {
    extern __shared__ uint8_t raw[];
    using S = FewShared<COLS>;
    constexpr int kStages = S::kStages;
    constexpr int kColumns = 2 * COLS < 32 ? 32 : 2 * COLS;
    S& s = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)tc::cluster_rank(), parts = p.splits;
    const int blocks = (int)((p.k + kTileK - 1) / kTileK);
    const int n0 = (int)(blockIdx.x / parts) * kRows;
    const int begin = (int)((int64_t)rank * blocks / parts), end = (int)((int64_t)(rank + 1) * blocks / parts);

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            bulk::barrier_init(&s.full[i], 1);
            bulk::barrier_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            bulk::barrier_init(&s.acc_full[i], 1);
            bulk::barrier_init(&s.acc_empty[i], 4);
        }
        bulk::barrier_init(&s.drained, 1);
        s.gave_up = 0;
        s.issued = 0;
        bulk::barrier_init_fence();
    }
    if (threadIdx.x == 4 * 32) {
        tc::prefetch_map(&map_a);
        tc::prefetch_map(&map_b);
    }
    if (warp == 5) tc::alloc<1>(&s.tensor_memory, kColumns);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *(volatile uint32_t*)&s.tensor_memory;
    volatile int* gave_up = &s.gave_up;

    if (warp == 4) {
        if (lane == 0) {
            int count = 0;
            for (int kb = begin; kb < end && count != p.copies[0]; ++kb, ++count) {
                const int stage = count % kStages;
                if (!tc::wait(&s.empty[stage], (count / kStages & 1) ^ 1, gave_up)) break;
                bulk::arrive_expect(&s.full[stage], (kRows + COLS) * kTileK);
                tc::load_tile(s.b[stage], &map_b, kb * kTileK, n0, &s.full[stage]);
                tc::load_tile(s.a[stage], &map_a, kb * kTileK, 0, &s.full[stage]);
            }
            s.issued = count;
        }
    } else if (warp == 5) {
        if (lane == 0) {
            constexpr uint32_t word = tc::instruction(kRows, COLS);
            int count = 0;
            for (int kb = begin; kb < end; ++kb, ++count) {
                const int stage = count % kStages, buffer = count & 1;
                if (!tc::wait(&s.acc_empty[buffer], (count >> 1 & 1) ^ 1, gave_up)) break;
                if (!tc::wait(&s.full[stage], count / kStages & 1, gave_up)) break;
                tc::fence_after();
                const uint64_t b = tc::operand(s.b[stage]), a = tc::operand(s.a[stage]);
#pragma unroll
                for (int k = 0; k < 4; ++k) tc::mma<1>(tmem + buffer * COLS, b + 2 * k, a + 2 * k, word, k > 0);
                tc::commit<1>(&s.empty[stage]);
                tc::commit<1>(&s.acc_full[buffer]);
            }
            if (*gave_up) {
                tc::commit<1>(&s.drained);
                bulk::wait(&s.drained, 0);
            }
        }
    } else {
        const int64_t n = n0 + threadIdx.x;
        const float* sb = p.b_scales + min(n, p.n - 1) / (p.b_tiles ? kBlock : 1) * p.b_scale_stride;
        const bool vec_a = p.a_scale_stride % 4 == 0 && reinterpret_cast<uintptr_t>(p.a_scales) % 16 == 0;
        const bool vec_b = p.b_scale_stride % 4 == 0 && reinterpret_cast<uintptr_t>(p.b_scales) % 16 == 0;
        const bool loader = threadIdx.x < COLS;
        const float* sa = p.a_scales + min((int64_t)threadIdx.x, p.m - 1) * p.a_scale_stride;
        uint64_t acc[COLS / 2];
#pragma unroll
        for (int i = 0; i < COLS / 2; ++i) acc[i] = 0;
        float4 next_b = scales4(sb, begin & ~3, end, vec_b), scale = next_b;
        float4 next_a = loader ? scales4(sa, begin & ~3, end, vec_a) : scale;
        int count = 0;
        for (int kb = begin; kb < end; ++kb, ++count) {
            const int buffer = count & 1, group = kb >> 2 & 1;
            if (kb == begin || (kb & 3) == 0) {
                scale = next_b;
                if (loader) {
                    s.a_scale[group][0][threadIdx.x] = next_a.x;
                    s.a_scale[group][1][threadIdx.x] = next_a.y;
                    s.a_scale[group][2][threadIdx.x] = next_a.z;
                    s.a_scale[group][3][threadIdx.x] = next_a.w;
                    next_a = scales4(sa, (kb & ~3) + 4, end, vec_a);
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                next_b = scales4(sb, (kb & ~3) + 4, end, vec_b);
            }
            const float mine = pick(scale, kb & 3);
            const uint64_t mine2 = tc::pair_of(mine, mine);
            tc::wait(&s.acc_full[buffer], count >> 1 & 1, gave_up);
            __syncwarp();
            tc::fence_after();
            const uint32_t from = tmem + ((uint32_t)(warp * 32) << 16) + buffer * COLS;
            constexpr int kStep = COLS < 32 ? COLS : 32;
#pragma unroll
            for (int c = 0; c < COLS; c += kStep) {
                uint32_t part[kStep];
                tc::load(from + c, part);
                tc::wait_loads();
                if (c + kStep == COLS) {
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tc::arrive(&s.acc_empty[buffer]);
                }
                const ulonglong2* sa2 = reinterpret_cast<const ulonglong2*>(&s.a_scale[group][kb & 3][c]);
#pragma unroll
                for (int i = 0; i < kStep / 2; i += 2) {
                    const ulonglong2 q = sa2[i / 2];
                    acc[c / 2 + i] =
                        tc::fma2(tc::pair_of(__uint_as_float(part[2 * i]), __uint_as_float(part[2 * i + 1])),
                                 tc::mul2(mine2, q.x), acc[c / 2 + i]);
                    acc[c / 2 + i + 1] =
                        tc::fma2(tc::pair_of(__uint_as_float(part[2 * i + 2]), __uint_as_float(part[2 * i + 3])),
                                 tc::mul2(mine2, q.y), acc[c / 2 + i + 1]);
                }
            }
        }
        if (tc::any_of(1, kRows, *gave_up)) {
#pragma unroll
            for (int i = 0; i < COLS / 2; ++i) acc[i] = ~uint64_t(0);  // two NaN
        }
        if (parts == 1) {
            OUT* q = static_cast<OUT*>(p.out) + n;
            if (n < p.n) {
#pragma unroll
                for (int i = 0; i < COLS / 2; ++i) {
                    float f[2];
                    tc::split_pair(acc[i], f[0], f[1]);
#pragma unroll
                    for (int j = 0; j < 2; ++j, q += p.out_stride)
                        if (2 * i + j < (int)p.m) *q = from_float<OUT>(p.accumulate ? to_float(*q) + f[j] : f[j]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < COLS / 2; ++i) {
                float x, y;
                tc::split_pair(acc[i], x, y);
                s.sum[2 * i][threadIdx.x] = x;
                s.sum[2 * i + 1][threadIdx.x] = y;
            }
        }
    }

    __syncthreads();
    if (*gave_up && threadIdx.x == 0) {
        atomicOr(&g_gave_up, 1u);
        for (int i = max(0, s.issued - kStages); i < s.issued; ++i) bulk::wait(&s.full[i % kStages], i / kStages & 1);
    }
    tc::cluster_sync();
    const int64_t n = n0 + threadIdx.x;
    if (parts > 1 && threadIdx.x < kRows && n < p.n) {
        OUT* const out = static_cast<OUT*>(p.out) + n;
        constexpr int kTogether = 8;  // rows whose sums are read at the same time
        for (int j0 = rank; j0 < (int)p.m; j0 += kTogether * parts) {
            float sum[kTogether];
#pragma unroll
            for (int i = 0; i < kTogether; ++i) sum[i] = 0.0f;
            for (int r = 0; r < parts; ++r) {
#pragma unroll
                for (int i = 0; i < kTogether; ++i) {
                    const int j = min(j0 + i * parts, COLS - 1);
                    sum[i] += tc::load_shared_at(tc::map_shared(&s.sum[j][threadIdx.x], r));
                }
            }
#pragma unroll
            for (int i = 0; i < kTogether; ++i) {
                const int j = j0 + i * parts;
                if (j < (int)p.m) {
                    OUT* q = out + j * p.out_stride;
                    *q = from_float<OUT>(p.accumulate ? to_float(*q) + sum[i] : sum[i]);
                }
            }
        }
    }
    tc::cluster_sync();  // the others may still read this CTA's sums
    if (warp == 5) tc::dealloc<1>(tmem, kColumns);
}

// ------------------------------------------------------------ host

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static const EncodeTiled f = [] {
        void* entry = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000, cudaEnableDefault, &found) !=
                cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            entry = nullptr;
        return reinterpret_cast<EncodeTiled>(entry);
    }();
    if (!f) raise(MDSOAP_DEVICE_UNAVAILABLE, "readout: the driver has no tensor maps");
    return f;
}

// Pieces of 128 bytes x `box_rows` rows of a matrix, swizzled in shared memory.
CUtensorMap tile_map(CUtensorMapDataType type, int size, const void* base, int64_t rows, int64_t cols, int64_t stride,
                     int box_rows) {
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)std::max<int64_t>(stride * size, 16)};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows}, steps[2] = {1, 1};
    if (encoder()(&map, type, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        raise(MDSOAP_INVALID_ARGUMENT, "readout: a product's operand cannot be described to the copy engine");
    return map;
}
CUtensorMap code_map(const void* base, int64_t rows, int64_t k, int64_t stride, int box_rows) {
    return tile_map(CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, rows, k, stride, box_rows);
}

// KERNEL is a template argument, so that each kernel has its own record of the
// devices where its shared memory limit is raised.
template <auto KERNEL, class... Args>
void launch(unsigned grid, unsigned cluster, unsigned threads, size_t bytes, int device, cudaStream_t stream,
            const Args&... args) {
    static std::atomic<uint64_t> done;
    allow_shared(KERNEL, (int)bytes, done, device, "product shared memory");
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = cluster;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = bytes;
    config.stream = stream;
    config.attrs = &attribute;
    config.numAttrs = 1;
    check(cudaLaunchKernelEx(&config, KERNEL, args...), "product launch");
}

// Blocks that a pair's first and second CTA copy at most (low and high half); the probe's.
std::atomic<uint64_t> g_copies{~uint64_t(0)};

// What a product of this shape runs.
struct Shape {
    bool few;
    int columns;  // few rows: A's rows, padded
    int splits;
    int64_t tiles;
    int64_t bytes;
};

Shape shape_of(int64_t m, int64_t n, int64_t k, int sms) {
    Shape s{};
    const int64_t blocks = blocks_of(k);
    s.few = m <= kRows;
    s.splits = 1;
    if (s.few) {
        s.columns = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
        s.tiles = blocks_of(n);
        // up to eight CTAs (the portable cluster) share K while SMs are free and each keeps two blocks
        while (s.splits < 8 && s.tiles * s.splits * 2 <= sms && blocks >= s.splits * 4) s.splits *= 2;
        return s;
    }
    s.tiles = ((m + kPairTile - 1) / kPairTile) * ((n + kPairTile - 1) / kPairTile);
    // Parts of K where whole tiles leave pairs idle.  In units of one block's time: rounds of the busiest pair, each
    // with 6 blocks' time around its sum, and for more than one part a second kernel that takes about 10 blocks'
    // time and reads every part of every tile, 1/60 of a block's time each.
    need(s.tiles < (1 << 25), "readout: product too large");
    const int64_t pairs = sms / 2;
    double best = 0.0;
    for (int64_t parts = 1; parts <= 32 && (parts == 1 || blocks >= parts * 4); ++parts) {
        const double rounds = (double)((s.tiles * parts + pairs - 1) / pairs);
        const double time = rounds * ((double)((blocks + parts - 1) / parts) + 6.0) +
                            (parts > 1 ? 10.0 + (double)(s.tiles * parts) / 60.0 : 0.0);
        if (parts == 1 || time < best) best = time, s.splits = (int)parts;
    }
    if (s.splits > 1) s.bytes = s.tiles * s.splits * kPairTile * kPairTile * (int64_t)sizeof(float);
    return s;
}

template <int COLS, class OUT>
void run_few(const void* a, int64_t a_stride, const void* b, int64_t b_stride, const ProductArgs& p, const Shape& s,
             int device, cudaStream_t stream) {
    const CUtensorMap map_a = code_map(a, p.m, p.k, a_stride, COLS), map_b = code_map(b, p.n, p.k, b_stride, kRows);
    launch<few_product_kernel<COLS, OUT>>((unsigned)(s.tiles * s.splits), (unsigned)s.splits, kFewThreads,
                                          sizeof(FewShared<COLS>) + 1024, device, stream, map_a, map_b, p);
}

template <bool TILES, class OUT>
void run_pairs(const void* a, int64_t a_stride, const void* b, int64_t b_stride, const ProductArgs& p, const Shape& s,
               int sms, int device, cudaStream_t stream) {
    const CUtensorMap map_a = code_map(a, p.m, p.k, a_stride, kRows), map_b = code_map(b, p.n, p.k, b_stride, kRows);
    const unsigned grid = 2 * (unsigned)std::min<int64_t>(sms / 2, s.tiles * s.splits);
    const size_t bytes = sizeof(PairShared<TILES>) + 1024;
    if (s.splits > 1) {
        const CUtensorMap map_parts = tile_map(CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, p.partials, s.tiles * s.splits * kPairTile,
                                               kPairTile, kPairTile, 32);
        launch<pair_product_kernel<TILES, float, Store::Partial>>(grid, 2, kThreads, bytes, device, stream, map_a, map_b, map_parts, p);
        // four rows a block; the grid holds 65 535 of them, and taller products go on from there
        const dim3 add((unsigned)((p.n + 255) / 256), (unsigned)std::min<int64_t>(65535, (p.m + 3) / 4));
        add_parts_kernel<OUT><<<add, 256, 0, stream>>>(p);
        check(cudaGetLastError(), "product launch");
    } else if (!p.accumulate && reinterpret_cast<uintptr_t>(p.out) % 16 == 0 &&
               (p.out_stride * sizeof(OUT)) % 16 == 0 && (p.n * sizeof(OUT)) % 16 == 0) {
        // the copy engine cuts rows off at whole 16 bytes: in a view whose rows end inside such a piece it would write
        // over what lies behind them
        const CUtensorMap map_out =
            tile_map(sizeof(OUT) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, sizeof(OUT),
                     p.out, p.m, p.n, p.out_stride, 32);
        launch<pair_product_kernel<TILES, OUT, Store::Tile>>(grid, 2, kThreads, bytes, device, stream, map_a, map_b, map_out, p);
    } else {
        launch<pair_product_kernel<TILES, OUT, Store::Direct>>(grid, 2, kThreads, bytes, device, stream, map_a, map_b, map_a, p);
    }
}

template <class OUT>
void run_product(const void* a, int64_t a_stride, const void* b, int64_t b_stride, const ProductArgs& p, const Shape& s,
                 int sms, int device, cudaStream_t stream) {
    if (s.few) {
        switch (s.columns) {
            case 16: run_few<16, OUT>(a, a_stride, b, b_stride, p, s, device, stream); break;
            case 32: run_few<32, OUT>(a, a_stride, b, b_stride, p, s, device, stream); break;
            case 64: run_few<64, OUT>(a, a_stride, b, b_stride, p, s, device, stream); break;
            default: run_few<128, OUT>(a, a_stride, b, b_stride, p, s, device, stream); break;
        }
    } else if (p.b_tiles) {
        run_pairs<true, OUT>(a, a_stride, b, b_stride, p, s, sms, device, stream);
    } else {
        run_pairs<false, OUT>(a, a_stride, b, b_stride, p, s, sms, device, stream);
    }
}

}  // namespace

extern "C" {

int mdsoap_matmul_bytes(int64_t m, int64_t n, int64_t k, int32_t b_tiles, int32_t device, int64_t* bytes) {
    return entry([&] {
        need(m >= 0 && n >= 0 && k >= 0 && bytes, "readout: invalid product shape");
        (void)b_tiles;  // the same work for both forms
        *bytes = m == 0 || n == 0 || k == 0 ? 0 : shape_of(m, n, k, sm_count(device)).bytes;
    });
}

int mdsoap_matmul(const void* a, int64_t m, int64_t a_stride, const float* a_scales, int64_t a_scale_stride,
                  const void* b, int64_t n, int64_t b_stride, const float* b_scales, int64_t b_scale_stride,
                  int32_t b_tiles, int64_t k, int32_t out_dtype, int32_t accumulate, void* out, int64_t out_stride,
                  void* workspace, int64_t workspace_bytes, int32_t device, void* stream) {
    return entry([&] {
        const int64_t limit = int64_t(1) << 30;
        need(m >= 0 && n >= 0 && k >= 0 && m < limit && n < limit && k < limit, "readout: invalid product shape");
        need(out_dtype == MDSOAP_FLOAT32 || out_dtype == MDSOAP_BFLOAT16,
             "readout: a product's type must be float32 or bfloat16");
        need(!accumulate || out_dtype == MDSOAP_FLOAT32, "readout: only a float32 product can be added to");
        if (m == 0 || n == 0) return;
        need(out && out_stride >= (m > 1 ? n : 0), "readout: invalid product output");
        const auto operand_ok = [&](const void* q, int64_t rows, int64_t stride, const float* scales, int64_t pitch) {
            return q && scales && reinterpret_cast<uintptr_t>(q) % 16 == 0 && stride % 16 == 0 &&
                   (rows <= 1 || (stride >= k && pitch >= blocks_of(k)));
        };
        need(k == 0 || (operand_ok(a, m, a_stride, a_scales, a_scale_stride) &&
                  operand_ok(b, n, b_stride, b_scales, b_tiles && n <= kBlock ? blocks_of(k) : b_scale_stride)),
             "readout: a product's operands need a 16-byte aligned base, a pitch that is a multiple of 16 and a scale "
             "for each block of 128");
        const OnDevice current(device);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const size_t size = out_dtype == MDSOAP_FLOAT32 ? 4 : 2;
        if (k == 0) {
            if (!accumulate) check(cudaMemset2DAsync(out, std::max(out_stride, n) * size, 0, n * size, m, s), "clear");
            return;
        }
        const int sms = sm_count(device);
        const Shape shape = shape_of(m, n, k, sms);
        need(shape.bytes == 0 || (workspace && workspace_bytes >= shape.bytes &&
                                  reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
             "readout: product workspace too small or not 16-byte aligned");
        ProductArgs p{m, n, k, a_scales, a_scale_stride, b_scales, b_scale_stride, b_tiles, out, out_stride, accumulate};
        p.splits = shape.splits;
        const uint64_t copies = g_copies.load(std::memory_order_relaxed);
        p.copies[0] = (int32_t)copies;
        p.copies[1] = (int32_t)(copies >> 32);
        p.partials = static_cast<float*>(workspace);
        if (out_dtype == MDSOAP_FLOAT32) run_product<float>(a, a_stride, b, b_stride, p, shape, sms, device, s);
        else run_product<__nv_bfloat16>(a, a_stride, b, b_stride, p, shape, sms, device, s);
    });
}

int mdsoap_matmul_check(int32_t device, void* stream) {
    return entry([&] {
        const OnDevice current(device);
        check(cudaStreamSynchronize(static_cast<cudaStream_t>(stream)), "stream sync");
        unsigned bits = 0;
        check(cudaMemcpyFromSymbol(&bits, g_gave_up, sizeof(bits)), "read product error word");
        if (!bits) return;
        const unsigned zero = 0;
        check(cudaMemcpyToSymbol(g_gave_up, &zero, sizeof(zero)), "clear product error word");
        raise(MDSOAP_INTERNAL, "product: copies or matrix instructions did not complete in time");
    });
}

void mdsoap_probe_matmul(int32_t first, int32_t second) {
    g_copies.store((uint64_t)(uint32_t)second << 32 | (uint32_t)first, std::memory_order_relaxed);
}

}  // extern "C"
