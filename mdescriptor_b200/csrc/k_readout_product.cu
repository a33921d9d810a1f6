// Product of two 8-bit matrices with scales for blocks of 128 on the tensor
// cores, and its C entry points (include/mdsoap.h).
#include "readout_host.cuh"
#include "tcgen05.cuh"

#include <algorithm>

using namespace mdsoap;
using namespace mdsoap::readout;

namespace {

constexpr int kTileM = 128;
constexpr int kTileK = 128;  // bytes of K a stage: one scale block
constexpr int kStages = 6;
constexpr int kPromote = 8;                       // warps that scale and add the partial products
constexpr int kThreads = (kPromote + 2) * 32;     // and one each for the copies and the matrix instructions

__device__ unsigned g_gave_up;  // products whose copies or matrix instructions did not complete in time

struct ProductArgs {
    int64_t m, n, k;
    const float* a_scales;
    int64_t a_scale_stride;
    const float* b_scales;
    int64_t b_scale_stride;
    void* out;
    int64_t out_stride;
    int32_t accumulate;
};

template <int BN>
struct Shared {
    uint8_t a[kStages][kTileM * kTileK];
    uint8_t b[kStages][BN * kTileK];
    float b_scale[2][BN];
    uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], drained;
    uint32_t tensor_memory;
    int gave_up;
    int issued;
};

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

// One CTA a tile of 128 x BN.  One thread copies tiles of A and B (one block of
// 128 of K a stage) into swizzled shared memory, one issues the matrix
// instructions of a block into one of two accumulators in tensor memory, and
// eight warps take each block's partial product out, multiply it by its scales
// and add it in float32 registers, while the other accumulator fills.
template <int BN, bool TILES, class OUT>
__global__ __launch_bounds__(kThreads, 1) void product_kernel(const __grid_constant__ CUtensorMap map_a,
                                                              const __grid_constant__ CUtensorMap map_b,
                                                              const __grid_constant__ ProductArgs p) {
    extern __shared__ __align__(1024) uint8_t raw[];
    Shared<BN>& s = *reinterpret_cast<Shared<BN>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    constexpr int kColumns = 2 * BN;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t m0 = (int64_t)blockIdx.y * kTileM, n0 = (int64_t)blockIdx.x * BN;
    const int blocks = (int)((p.k + kTileK - 1) / kTileK);

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            bulk::barrier_init(&s.full[i], 1);
            bulk::barrier_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            bulk::barrier_init(&s.acc_full[i], 1);
            bulk::barrier_init(&s.acc_empty[i], kPromote);
        }
        bulk::barrier_init(&s.drained, 1);
        s.gave_up = 0;
        s.issued = 0;
        bulk::barrier_init_fence();
    }
    if (warp == kPromote + 1) tc::alloc(&s.tensor_memory, kColumns);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *(volatile uint32_t*)&s.tensor_memory;
    volatile int* gave_up = &s.gave_up;

    if (warp == kPromote) {
        if (lane == 0) {
            int kb = 0;
            for (; kb < blocks; ++kb) {
                const int stage = kb % kStages;
                if (!tc::wait(&s.empty[stage], (kb / kStages & 1) ^ 1, gave_up)) break;
                bulk::arrive_expect(&s.full[stage], (kTileM + BN) * kTileK);
                tc::load_tile(s.a[stage], &map_a, kb * kTileK, (int)m0, &s.full[stage]);
                tc::load_tile(s.b[stage], &map_b, kb * kTileK, (int)n0, &s.full[stage]);
            }
            s.issued = kb;
        }
    } else if (warp == kPromote + 1) {
        if (lane == 0) {
            constexpr uint32_t word = tc::instruction(kTileM, BN);
            for (int kb = 0; kb < blocks; ++kb) {
                const int stage = kb % kStages, buffer = kb & 1;
                if (!tc::wait(&s.acc_empty[buffer], (kb >> 1 & 1) ^ 1, gave_up)) break;
                if (!tc::wait(&s.full[stage], kb / kStages & 1, gave_up)) break;
                tc::fence_after();
                const uint64_t a = tc::operand(s.a[stage]), b = tc::operand(s.b[stage]);
#pragma unroll
                for (int k = 0; k < 4; ++k) tc::mma(tmem + buffer * BN, a + 2 * k, b + 2 * k, word, k > 0);
                tc::commit(&s.empty[stage]);
                tc::commit(&s.acc_full[buffer]);
            }
            if (*gave_up) {  // matrix instructions in flight end before the tensor memory goes
                tc::commit(&s.drained);
                bulk::wait(&s.drained, 0);
            }
        }
    } else {
        constexpr int kMine = BN / 2;  // columns of one thread
        const int quarter = warp & 3, half = warp >> 2;
        const int64_t row = m0 + quarter * 32 + lane;
        const int64_t col = n0 + half * kMine;
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + half * kMine;
        float acc[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) acc[i] = 0.0f;
        const bool live = row < p.m;
        const float* sa = p.a_scales + (live ? row : 0) * p.a_scale_stride;
        const int64_t b_row = TILES ? min(col, p.n - 1) / kBlock : n0 + threadIdx.x;
        const bool b_live = TILES || (threadIdx.x < BN && b_row < p.n);
        const float* sb = p.b_scales + (b_live ? b_row : 0) * p.b_scale_stride;
        float next_a = live && blocks ? sa[0] : 0.0f, next_b = b_live && blocks ? sb[0] : 0.0f;
        for (int kb = 0; kb < blocks; ++kb) {
            const int buffer = kb & 1;
            const float scale_a = next_a, scale_b = next_b;
            if (kb + 1 < blocks) {
                if (live) next_a = sa[kb + 1];
                if (b_live) next_b = sb[kb + 1];
            }
            if constexpr (!TILES) {
                if (threadIdx.x < BN) s.b_scale[buffer][threadIdx.x] = scale_b;
                asm volatile("bar.sync 1, %0;" ::"n"(kPromote * 32) : "memory");
            }
            if (!tc::wait(&s.acc_full[buffer], kb >> 1 & 1, gave_up)) *gave_up = 1;
            __syncwarp();
            tc::fence_after();
#pragma unroll
            for (int c = 0; c < kMine; c += 32) {
                uint32_t part[32];
                tc::load32(from + buffer * BN + c, part);
                tc::wait_loads();
                if (c + 32 == kMine) {
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tc::arrive(&s.acc_empty[buffer]);
                }
                if constexpr (TILES) {
                    const float scale = scale_a * scale_b;
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc[c + i] = fmaf(__uint_as_float(part[i]), scale, acc[c + i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        acc[c + i] = fmaf(__uint_as_float(part[i]), scale_a * s.b_scale[buffer][half * kMine + c + i],
                                          acc[c + i]);
                }
            }
        }
        if (live && !*gave_up)
            store_row(static_cast<OUT*>(p.out) + row * p.out_stride + col, p.n - col, acc, p.accumulate);
    }

    __syncthreads();
    if (*gave_up && threadIdx.x == 0) {
        atomicOr(&g_gave_up, 1u);
        // copies in flight land before the shared memory goes
        for (int kb = max(0, s.issued - kStages); kb < s.issued; ++kb)
            bulk::wait(&s.full[kb % kStages], kb / kStages & 1);
    }
    __syncthreads();
    if (warp == kPromote + 1) tc::dealloc(tmem, kColumns);
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

CUtensorMap tile_map(const void* base, int64_t rows, int64_t k, int64_t stride, int box_rows) {
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)std::max<int64_t>(stride, 16)};
    const cuuint32_t box[2] = {kTileK, (cuuint32_t)box_rows}, steps[2] = {1, 1};
    if (encoder()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        raise(MDSOAP_INVALID_ARGUMENT, "readout: a product's operand cannot be described to the copy engine");
    return map;
}

template <int BN, bool TILES, class OUT>
void launch_product(const CUtensorMap& a, const CUtensorMap& b, const ProductArgs& p, cudaStream_t stream) {
    auto kernel = product_kernel<BN, TILES, OUT>;
    constexpr int bytes = sizeof(Shared<BN>) + 1024;
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "product shared memory");
    const dim3 grid((unsigned)((p.n + BN - 1) / BN), (unsigned)((p.m + kTileM - 1) / kTileM));
    kernel<<<grid, kThreads, bytes, stream>>>(a, b, p);
    check(cudaGetLastError(), "product launch");
}

}  // namespace

extern "C" {

int mdsoap_matmul_bytes(int64_t m, int64_t n, int64_t k, int32_t b_tiles, int32_t device, int64_t* bytes) {
    return entry([&] {
        need(m >= 0 && n >= 0 && k >= 0 && bytes, "readout: invalid product shape");
        (void)b_tiles;
        (void)device;
        *bytes = 0;
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
        check(cudaSetDevice(device), "cudaSetDevice");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const size_t size = out_dtype == MDSOAP_FLOAT32 ? 4 : 2;
        if (k == 0) {
            if (!accumulate) check(cudaMemset2DAsync(out, std::max(out_stride, n) * size, 0, n * size, m, s), "clear");
            return;
        }
        (void)workspace;
        (void)workspace_bytes;
        constexpr int BN = 128;
        need((m + kTileM - 1) / kTileM <= 65535, "readout: too many rows in a product");
        const CUtensorMap map_a = tile_map(a, m, k, a_stride, kTileM), map_b = tile_map(b, n, k, b_stride, BN);
        const ProductArgs p{m, n, k, a_scales, a_scale_stride, b_scales, b_scale_stride, out, out_stride, accumulate};
        if (out_dtype == MDSOAP_FLOAT32) {
            if (b_tiles) launch_product<BN, true, float>(map_a, map_b, p, s);
            else launch_product<BN, false, float>(map_a, map_b, p, s);
        } else {
            if (b_tiles) launch_product<BN, true, __nv_bfloat16>(map_a, map_b, p, s);
            else launch_product<BN, false, __nv_bfloat16>(map_a, map_b, p, s);
        }
    });
}

int mdsoap_matmul_check(int32_t device, void* stream) {
    return entry([&] {
        check(cudaSetDevice(device), "cudaSetDevice");
        check(cudaStreamSynchronize(static_cast<cudaStream_t>(stream)), "stream sync");
        unsigned bits = 0;
        check(cudaMemcpyFromSymbol(&bits, g_gave_up, sizeof(bits)), "read product error word");
        if (!bits) return;
        const unsigned zero = 0;
        check(cudaMemcpyToSymbol(g_gave_up, &zero, sizeof(zero)), "clear product error word");
        raise(MDSOAP_INTERNAL, "product: copies or matrix instructions did not complete in time");
    });
}

}  // extern "C"
