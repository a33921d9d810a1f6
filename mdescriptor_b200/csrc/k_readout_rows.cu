// Readout operators on rows: root-mean-square norm with the residual's
// addition (wide or 8-bit output), its gradient, and the 8-bit block
// quantiser, with their C entry points (include/mdsoap.h).
#include "host_errors.cuh"
#include "readout.cuh"
#include "readout_host.cuh"
#include "bulk_copy.cuh"

#include <algorithm>

using namespace mdsoap;
using namespace mdsoap::readout;

namespace {

constexpr int kRowWarps = 8;  // warps per CTA of the row kernel

enum class Rows { Norm8, NormWide, Quantize };

template <class T>
struct RowArgs {
    MatrixIn<T> x;
    const T* residual;
    int64_t residual_stride;
    const float* col_factor;  // norm weight, or the quantiser's column factor; may be null
    const float* row_factor;  // quantiser only; may be null
    float eps;
    T* sum;
    int64_t sum_stride;
    float* rstd;
    T* wide;
    int64_t wide_stride;
    uint8_t* codes;
    int64_t code_stride;
    float* scales;
    int64_t scale_stride;
};

// One row by one warp (CTA_ROW false) or by the CTA's warps together, a block
// of 128 at a time, four elements a lane.
//
// s = x + r; rstd = (mean s^2 + eps)^-1/2; y = s rstd w.  In 8 bits the factor
// rstd is constant in the row, so it cancels from the codes 448 z / max|z| of
// z = s w and lives in the scales alone: the codes are written in the one pass
// that also sums s^2, and only the blocks' maxima wait for the row's end (in
// shared memory, one float a block).  Nothing of the row is held or read twice.
// Bound by HBM: x and r once in, sum and codes once out.  131 072 x 2100 bfloat16
// rows with residual: 321 us a pass, 6.0 TB/s (302 us and 1.91 GB of DRAM traffic
// for the kernel alone, 56 % of issue slots used); with 16-byte units, two blocks
// a warp and the maxima by shuffles it took 593 us, 54 instructions an element.
template <class T, bool CTA_ROW, Rows MODE>
struct RowPass {
    using Word = typename Quad<T>::Word;
    static constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;
    static constexpr int kStep = CTA_ROW ? kRowWarps : 1;  // blocks from one of a warp's to its next
    const RowArgs<T>& a;
    const T* x;
    const T* r;  // null without a residual
    T* sum;      // null where it is not wanted
    uint8_t* codes;
    float* top;
    int width;
    uintptr_t x_begin, x_end, r_begin, r_end;
    float total;

    // One whole block from its words.  ALIGNED: rows and factors can be read and written in words.
    template <bool ALIGNED>
    __device__ __forceinline__ void block(int col, const Word& wx, const Word& wr) {
        const int lane = threadIdx.x & 31;
        float4 s = unpack4<T>(wx);
        if (r) {
            const float4 f = unpack4<T>(wr);
            s.x += f.x, s.y += f.y, s.z += f.z, s.w += f.w;
        }
        if constexpr (MODE != Rows::Quantize) {
            total = fmaf(s.x, s.x, fmaf(s.y, s.y, fmaf(s.z, s.z, fmaf(s.w, s.w, total))));
            if (sum) {
                if constexpr (ALIGNED) *reinterpret_cast<Word*>(sum + col) = pack4<T>(s);
                else store_quad(sum, col, width, pack4<T>(s));
            }
        }
        if constexpr (MODE != Rows::NormWide) {
            float4 z = s;
            if (MODE == Rows::Norm8 || a.col_factor) {
                float4 w;
                if constexpr (ALIGNED) {
                    w = __ldg(reinterpret_cast<const float4*>(a.col_factor + col));
                } else {
                    float f[4];
                    load_vector<4>(a.col_factor, col, width, f);
                    w = make_float4(f[0], f[1], f[2], f[3]);
                }
                z = make_float4(s.x * w.x, s.y * w.y, s.z * w.z, s.w * w.w);
            }
            const float most = warp_larger(larger(larger(z.x, z.y, z.z), z.w));
            const Factor factor(most);
            if (lane == 0) top[col / kBlock] = most;
            *reinterpret_cast<uint32_t*>(codes + col) = codes4(factor(z.x), factor(z.y), factor(z.z), factor(z.w));
        }
    }

    // kAhead blocks from `b` on, their words loaded first.
    template <bool ALIGNED>
    __device__ __forceinline__ void several(int b) {
        const int col = b * kBlock + (int)(threadIdx.x & 31) * 4;
        Word wx[kAhead], wr[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const T* px = x + col + i * kStep * kBlock;
            const T* pr = r + col + i * kStep * kBlock;
            wx[i] = ALIGNED ? __ldg(reinterpret_cast<const Word*>(px)) : load_split(px);
            if (r) wr[i] = ALIGNED ? __ldg(reinterpret_cast<const Word*>(pr)) : load_split(pr);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) block<ALIGNED>(col + i * kStep * kBlock, wx[i], wr[i]);
    }

    // One block element by element, a lane every 32nd, each access of the warp a run of neighbouring ones: the last
    // of a row, and what is left over.
    __device__ __forceinline__ void scattered(int b) {
        const int lane = threadIdx.x & 31, col = b * kBlock + lane;
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool live = col + 32 * i < width;
            s[i] = live ? to_float(x[col + 32 * i]) : 0.0f;
            if (r && live) s[i] += to_float(r[col + 32 * i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool live = col + 32 * i < width;
            if constexpr (MODE != Rows::Quantize) {
                total = fmaf(s[i], s[i], total);
                if (sum && live) sum[col + 32 * i] = from_float<T>(s[i]);
            }
            if (MODE != Rows::NormWide && live && (MODE == Rows::Norm8 || a.col_factor))
                s[i] *= __ldg(a.col_factor + col + 32 * i);
        }
        if constexpr (MODE != Rows::NormWide) {
            const float most = warp_larger(larger(larger(s[0], s[1], s[2]), s[3]));
            const Factor factor(most);
            if (lane == 0) top[b] = most;
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const uint32_t q = codes2(factor(s[i]), factor(s[i + 1]));
                if (col + 32 * i < width) codes[col + 32 * i] = (uint8_t)q;
                if (col + 32 * i + 32 < width) codes[col + 32 * i + 32] = (uint8_t)(q >> 8);
            }
        }
    }

    // Whether the aligned words around columns [0, columns) of a row lie inside its matrix.
    __device__ __forceinline__ bool inside(const T* row, int columns, uintptr_t begin, uintptr_t end) const {
        const uintptr_t at = reinterpret_cast<uintptr_t>(row), shift = at % sizeof(Word);
        return shift == 0 || (at - shift >= begin && at - shift + columns * sizeof(T) + sizeof(Word) <= end);
    }

    // The warp's blocks: kAhead of them under way at a time.
    __device__ __forceinline__ void run(int first) {
        const int full = width / kBlock;
        int b = first;
        if (quads_aligned(x) && (!r || quads_aligned(r)) && (!sum || quads_aligned(sum)) &&
            reinterpret_cast<uintptr_t>(a.col_factor) % 16 == 0) {
            for (; b + (kAhead - 1) * kStep < full; b += kAhead * kStep) several<true>(b);
            for (; b < full; b += kStep) {
                const int col = b * kBlock + (int)(threadIdx.x & 31) * 4;
                block<true>(col, __ldg(reinterpret_cast<const Word*>(x + col)),
                            r ? __ldg(reinterpret_cast<const Word*>(r + col)) : Word{});
            }
        } else if (inside(x, full * kBlock, x_begin, x_end) && (!r || inside(r, full * kBlock, r_begin, r_end))) {
            for (; b + (kAhead - 1) * kStep < full; b += kAhead * kStep) several<false>(b);
        }
        for (; b * kBlock < width; b += kStep) scattered(b);
    }
};

template <class T, bool CTA_ROW, Rows MODE>
__global__ __launch_bounds__(kRowWarps * 32, 4) void rows_kernel(const __grid_constant__ RowArgs<T> a) {
    extern __shared__ float s_top[];
    __shared__ float s_sum[kRowWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = CTA_ROW ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kRowWarps + warp;
    if (row >= a.x.rows) return;  // never with CTA_ROW, whose warps meet below
    const int64_t width = a.x.width;
    const int64_t nblocks = (width + kBlock - 1) / kBlock;
    const auto span_end = [&](const T* p, int64_t stride) {
        return reinterpret_cast<uintptr_t>(p + (a.x.rows - 1) * stride + width);
    };
    RowPass<T, CTA_ROW, MODE> pass{a,
                                   a.x.data + row * a.x.stride,
                                   a.residual ? a.residual + row * a.residual_stride : nullptr,
                                   MODE != Rows::Quantize && a.sum ? a.sum + row * a.sum_stride : nullptr,
                                   a.codes + row * a.code_stride,
                                   s_top + (CTA_ROW ? 0 : warp * nblocks),
                                   (int)width,
                                   reinterpret_cast<uintptr_t>(a.x.data), span_end(a.x.data, a.x.stride),
                                   reinterpret_cast<uintptr_t>(a.residual), span_end(a.residual, a.residual_stride),
                                   0.0f};
    const int first = CTA_ROW ? warp : 0, step = CTA_ROW ? kRowWarps : 1;
    pass.run(first);

    float row_scale = 1.0f;
    if constexpr (MODE != Rows::Quantize) {
        float total = warp_sum(pass.total);
        if constexpr (CTA_ROW) {
            if (lane == 0) s_sum[warp] = total;
            __syncthreads();
            total = 0.0f;
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) total += s_sum[w];
        }
        row_scale = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(total, (float)width) + a.eps));
        if (a.rstd && lane == 0 && (!CTA_ROW || warp == 0)) a.rstd[row] = row_scale;
    } else if (a.row_factor) {
        row_scale = a.row_factor[row];  // a negative one shows in the scales' sign
    }
    if constexpr (CTA_ROW) __syncthreads();
    __syncwarp();

    if constexpr (MODE == Rows::NormWide) {
        for (int64_t b = first; b < nblocks; b += step) {
            const int64_t col = b * kBlock + lane * 4;
            float4 s = unpack4<T>(load_quad(pass.x, col, width, pass.x_begin, pass.x_end));
            if (pass.r) {
                const float4 f = unpack4<T>(load_quad(pass.r, col, width, pass.r_begin, pass.r_end));
                s.x += f.x, s.y += f.y, s.z += f.z, s.w += f.w;
            }
            float w[4];
            load_vector<4>(a.col_factor, col, width, w);
            store_quad(a.wide + row * a.wide_stride, col, width,
                       pack4<T>(make_float4(s.x * row_scale * w[0], s.y * row_scale * w[1], s.z * row_scale * w[2],
                                            s.w * row_scale * w[3])));
        }
    } else {
        const int at = CTA_ROW ? threadIdx.x : lane;
        for (int64_t b = at; b < nblocks; b += CTA_ROW ? kRowWarps * 32 : 32)
            a.scales[row * a.scale_stride + b] = scale_of(pass.top[b]) * row_scale;
    }
}

template <class T, Rows MODE>
void launch_rows(const RowArgs<T>& a, int device, cudaStream_t stream) {
    if (a.x.rows == 0 || a.x.width == 0) return;
    const int sms = sm_count(device);
    const int64_t nblocks = blocks_of(a.x.width);
    const bool tops = MODE != Rows::NormWide;
    const size_t warp_bytes = tops ? nblocks * sizeof(float) : 0;
    constexpr int kMost = 200 * 1024;
    if (warp_bytes > kMost) raise(MDSOAP_INVALID_ARGUMENT, "readout rows: width exceeds 6 553 600 columns");
    // A warp a row keeps all reductions inside the warp; a CTA a row when there
    // are too few rows to fill the SMs that way, or the maxima of eight rows
    // would not fit.
    const bool cta_row = a.x.rows < (int64_t)sms * kRowWarps * 2 || warp_bytes * kRowWarps > 48 * 1024;
    if (cta_row) {
        auto kernel = rows_kernel<T, true, MODE>;
        // the 48 KB that every launch may have hold the kernel's own few bytes too; the limit is the kernel's, not the
        // launch's, so it is raised once and to the most that any width takes
        static std::atomic<uint64_t> done;
        if (warp_bytes > 40 * 1024) allow_shared(kernel, kMost, done, device, "readout rows: shared memory");
        if (a.x.rows > 0x7fffffff) raise(MDSOAP_INVALID_ARGUMENT, "readout rows: too many rows");
        kernel<<<(unsigned)a.x.rows, kRowWarps * 32, warp_bytes, stream>>>(a);
    } else {
        const int64_t grid = (a.x.rows + kRowWarps - 1) / kRowWarps;
        if (grid > 0x7fffffff) raise(MDSOAP_INVALID_ARGUMENT, "readout rows: too many rows");
        rows_kernel<T, false, MODE><<<(unsigned)grid, kRowWarps * 32, warp_bytes * kRowWarps, stream>>>(a);
    }
    check(cudaGetLastError(), "readout rows launch");
}

// ------------------------------------------------------------ norm gradient
//
// c = sum_d dy w s;  ds = rstd w dy - s rstd^3 c / D (+ dsum);  dw = sum_t dy s rstd.
//
// A CTA takes rows b, b + grid, ...: each thread owns the same NU units of 16
// bytes of every row.  Its units of the next kDepth - 1 rows are on their way
// into its own slots of a ring in shared memory (nobody else reads them, so no
// barrier guards them); a row stays in registers between the sum c and the
// result, and the weight's gradient adds up in registers over the CTA's rows.
// The partial sums of all CTAs go to the workspace and are added in CTA order by
// a second kernel: the same bits on every run.  Bound by HBM: dy, s, dsum once
// in, ds once out.
//
// ALIKE: the matrices' rows sit alike relative to 16 bytes.  With an odd width
// the rows' alignment repeats every eight rows at most; the grid is a multiple of
// that, so all rows of a CTA are aligned alike and its units are whole 16-byte
// words of all of them (the first and last of a row partly another row's).
//
// 40 001 x 2325 bfloat16 rows with dsum: 149 us a pass, 5.0 TB/s (142 us for this
// kernel, 7 for the sum of its partial results); spliced words and no ring took
// 802 us, aligned words 284, the ring 200.  What is left is its barrier a row.
template <class T>
struct NormBackwardArgs {
    MatrixIn<T> dy, s;
    const T* dsum;
    int64_t dsum_stride;
    const float* rstd;
    const float* weight;
    T* dx;
    int64_t dx_stride;
    float* partial;  // [grid][pitch]
    int64_t pitch;
    float* dots;  // wide rows only: c of each row
};

// The sum over the CTA's warps (at most 16); `scratch` holds zeros beyond theirs.
__device__ __forceinline__ float cta_sum(float x, float (&scratch)[16]) {
    x = warp_sum(x);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    float4 part[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) part[i] = reinterpret_cast<const float4*>(scratch)[i];
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) total += (part[i].x + part[i].y) + (part[i].z + part[i].w);
    return total;
}

__device__ __forceinline__ void copy16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(bulk::smem_u32(to)), "l"(from) : "memory");
}

__host__ __device__ constexpr int ring_depth(int units) { return units == 1 ? 4 : units == 2 ? 3 : 2; }

template <class T, int NU, bool ALIKE>
__global__ __launch_bounds__(512, NU == 1 ? 2 : 1) void norm_backward_kernel(const __grid_constant__ NormBackwardArgs<T> a) {
    constexpr int N = kUnit<T>;
    constexpr int kDepth = ring_depth(NU);
    constexpr bool kHeld = NU <= 2;  // the weight stays in registers
    extern __shared__ uint4 ring[];  // [kDepth][3][NU][threads]
    __shared__ __align__(16) float scratch[2][16];
    const int width = (int)a.s.width, threads = blockDim.x;
    const MatrixIn<T> dsum{a.dsum, a.s.rows, a.s.width, a.dsum_stride};
    const int64_t first = blockIdx.x;
    const int before = ALIKE ? (int)(reinterpret_cast<uintptr_t>(a.s.data + first * a.s.stride) % 16 / sizeof(T)) : 0;
    if (threadIdx.x < 32) scratch[threadIdx.x / 16][threadIdx.x % 16] = 0.0f;

    int col[NU];
    bool whole[NU];
    uint4 mask[NU];  // the bits of a unit that lie inside the row
    float w[kHeld ? NU : 1][N], dw[NU][N];
    const auto weight_of = [&](int u, float (&f)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = col[u] + i >= 0 && col[u] + i < width ? __ldg(a.weight + col[u] + i) : 0.0f;
    };
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        col[u] = (u * threads + threadIdx.x) * N - before;
        whole[u] = col[u] >= 0 && col[u] + N <= width;
        uint32_t bits[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col[u] + i >= 0 && col[u] + i < width)
                bits[i * 4 / N] |= (sizeof(T) == 4 ? 0xffffffffu : 0xffffu) << (sizeof(T) == 4 ? 0 : i % 2 * 16);
        mask[u] = make_uint4(bits[0], bits[1], bits[2], bits[3]);
        if constexpr (kHeld) weight_of(u, w[u]);
#pragma unroll
        for (int i = 0; i < N; ++i) dw[u][i] = 0.0f;
    }
    bool all_whole = true;  // of the warp's lanes and units
#pragma unroll
    for (int u = 0; u < NU; ++u) all_whole = all_whole && __all_sync(0xffffffffu, whole[u]);
    // Slots of dy, s and dsum of a stage follow each other, `threads` apart.
    const int span = 3 * NU * threads;
    uint4* const mine = ring + threadIdx.x;
    // One unit of a row into its slot; `p` is the unit's address.
    const auto fetch = [&](const MatrixIn<T>& m, const T* p, int64_t row, int u, uint4& to) {
        if constexpr (ALIKE) {
            if (whole[u]) {
                copy16(&to, p);
            } else if (col[u] < width && col[u] + N > 0) {
                if (p >= m.data && p + N <= m.data + (m.rows - 1) * m.stride + width) {
                    copy16(&to, p);
                    return;
                }
                uint4 q = make_uint4(0, 0, 0, 0);
                T* t = reinterpret_cast<T*>(&q);
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (col[u] + i >= 0 && col[u] + i < width) t[i] = p[i];
                to = q;
            }
        } else {
            to = m.unit(row, col[u]);
        }
    };
    // The row that is fetched next, and its addresses.
    int64_t ahead = first;
    const T *next_dy = a.dy.data + first * a.dy.stride, *next_s = a.s.data + first * a.s.stride,
            *next_d = a.dsum ? a.dsum + first * a.dsum_stride : nullptr;
    const int64_t step_dy = a.dy.stride * gridDim.x, step_s = a.s.stride * gridDim.x, step_d = a.dsum_stride * gridDim.x;
    const auto fetch_row = [&](uint4* to) {
        if (ahead < a.s.rows) {
            if (ALIKE && all_whole) {
#pragma unroll
                for (int u = 0; u < NU; ++u, to += 3 * threads) {
                    copy16(to, next_dy + col[u]);
                    copy16(to + threads, next_s + col[u]);
                    if (a.dsum) copy16(to + 2 * threads, next_d + col[u]);
                }
            } else {
#pragma unroll
                for (int u = 0; u < NU; ++u, to += 3 * threads) {
                    fetch(a.dy, next_dy + col[u], ahead, u, to[0]);
                    fetch(a.s, next_s + col[u], ahead, u, to[threads]);
                    if (a.dsum) fetch(dsum, next_d + col[u], ahead, u, to[2 * threads]);
                }
            }
        }
        ahead += gridDim.x, next_dy += step_dy, next_s += step_s, next_d += step_d;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // A unit's floats; zero outside the row.
    const auto take = [&](const uint4& q, int u, float (&f)[N]) {
        unpack<T>(make_uint4(q.x & mask[u].x, q.y & mask[u].y, q.z & mask[u].z, q.w & mask[u].w), f);
    };

    const float inv_width = __fdiv_rn(1.0f, (float)width);
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) fetch_row(mine + i * span);
    float next_rstd = first < a.s.rows ? a.rstd[first] : 0.0f;
    __syncthreads();  // the zeros of `scratch`
    int turn = 0;
    uint4 *now = mine, *behind = mine + (kDepth - 1) * span;  // the slots of this row and of the one before it
    T* dx = a.dx + first * a.dx_stride;
    for (int64_t row = first; row < a.s.rows; row += gridDim.x, dx += a.dx_stride * gridDim.x, turn ^= 1) {
        fetch_row(behind);
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
        const float rstd = next_rstd;
        if (row + gridDim.x < a.s.rows) next_rstd = a.rstd[row + gridDim.x];
        float dy[NU][N], s[NU][N];
        float c = 0.0f;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            float g[N];
            take(now[3 * u * threads], u, dy[u]);
            take(now[(3 * u + 1) * threads], u, s[u]);
            if constexpr (!kHeld) weight_of(u, g);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                dw[u][i] = fmaf(dy[u][i], s[u][i] * rstd, dw[u][i]);
                dy[u][i] *= kHeld ? w[kHeld ? u : 0][i] : g[i];
                c = fmaf(dy[u][i], s[u][i], c);
            }
        }
        // two scratch rows in turn: a warp may be one row ahead of another, never two
        c = cta_sum(c, scratch[turn]) * inv_width * rstd * rstd * rstd;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            float out[N];
            if (a.dsum) {
                unpack<T>(now[(3 * u + 2) * threads], out);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) out[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) out[i] = fmaf(-s[u][i], c, fmaf(dy[u][i], rstd, out[i]));
            if constexpr (ALIKE) {
                const uint4 q = pack<T>(out);
                if (all_whole || whole[u]) {
                    *reinterpret_cast<uint4*>(dx + col[u]) = q;
                } else if (col[u] < width && col[u] + N > 0) {
                    const T* t = reinterpret_cast<const T*>(&q);
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (col[u] + i >= 0 && col[u] + i < width) dx[col[u] + i] = t[i];
                }
            } else {
                store_unit(dx, col[u], width, pack<T>(out));
            }
        }
        behind = now;
        now = now == mine + (kDepth - 1) * span ? mine : now + span;
    }
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col[u] + i >= 0 && col[u] + i < width) a.partial[blockIdx.x * a.pitch + col[u] + i] = dw[u][i];
}

// Rows too wide for one CTA's registers: c of each row first ...
template <class T>
__global__ __launch_bounds__(256) void norm_dots_kernel(const __grid_constant__ NormBackwardArgs<T> a) {
    constexpr int N = kUnit<T>;
    __shared__ __align__(16) float scratch[16];
    if (threadIdx.x < 16) scratch[threadIdx.x] = 0.0f;
    __syncthreads();
    const int64_t row = blockIdx.x;
    float c = 0.0f;
    for (int64_t col = (int64_t)threadIdx.x * N; col < a.s.width; col += 256 * N) {
        float dy[N], s[N], w[N];
        unpack<T>(a.dy.unit(row, col), dy);
        unpack<T>(a.s.unit(row, col), s);
        load_vector<N>(a.weight, col, a.s.width, w);
#pragma unroll
        for (int i = 0; i < N; ++i) c = fmaf(dy[i] * w[i], s[i], c);
    }
    c = cta_sum(c, scratch);
    if (threadIdx.x == 0) a.dots[row] = c;
}

// ... then stripes of columns over ranges of rows.
template <class T>
__global__ __launch_bounds__(256) void norm_stripes_kernel(const __grid_constant__ NormBackwardArgs<T> a) {
    constexpr int N = kUnit<T>;
    const int64_t width = a.s.width;
    const MatrixIn<T> dsum{a.dsum, a.s.rows, width, a.dsum_stride};
    const int64_t col = ((int64_t)blockIdx.y * 256 + threadIdx.x) * N;
    const float inv_width = __fdiv_rn(1.0f, (float)width);
    float w[N], dw[N];
    load_vector<N>(a.weight, col, width, w);
#pragma unroll
    for (int i = 0; i < N; ++i) dw[i] = 0.0f;
    for (int64_t row = blockIdx.x; row < a.s.rows; row += gridDim.x) {
        const float rstd = a.rstd[row];
        const float c = a.dots[row] * inv_width * rstd * rstd;
        float dy[N], s[N], out[N];
        unpack<T>(a.dy.unit(row, col), dy);
        unpack<T>(a.s.unit(row, col), s);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            dw[i] = fmaf(dy[i], s[i] * rstd, dw[i]);
            out[i] = rstd * fmaf(-s[i], c, dy[i] * w[i]);
        }
        if (a.dsum) {
            float d[N];
            unpack<T>(dsum.unit(row, col), d);
#pragma unroll
            for (int i = 0; i < N; ++i) out[i] += d[i];
        }
        store_unit(a.dx + row * a.dx_stride, col, width, pack<T>(out));
    }
    if (col < width) {
        float4* p = reinterpret_cast<float4*>(a.partial + blockIdx.x * a.pitch + col);
#pragma unroll
        for (int i = 0; i < N; i += 4) p[i / 4] = make_float4(dw[i], dw[i + 1], dw[i + 2], dw[i + 3]);
    }
}

// dweight[d] = the CTAs' partial sums: 32 threads a column take every 32nd row
// of `partial` each, and their sums are added in order.
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* partial, int64_t pitch, int count, int64_t width,
                                                          float* out) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + lane;
    float total = 0.0f;
    if (col < width) {
#pragma unroll 8
        for (int b = part; b < count; b += 32) total += partial[b * pitch + col];
    }
    s[part][lane] = total;
    __syncthreads();
    if (part == 0 && col < width) {
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) total += s[i][lane];
        out[col] = total;
    }
}

struct BackwardShape {
    int threads, units;  // 0 threads: the two-kernel form
    int64_t grid, pitch;
    size_t bytes;
};

// Threads and units so that a row (and the word that an odd start adds) fits a
// CTA's registers, and a grid that the SMs hold at once: by registers, 64 a
// thread with one unit and 128 with more.
BackwardShape backward_shape(int64_t rows, int64_t width, int unit, int sms) {
    BackwardShape s{};
    s.pitch = (width + 7) / 8 * 8;
    const int64_t units = (width + unit - 1) / unit + 1;
    // two units a thread where a row has them: what a row costs beside its elements (its sum over the CTA, its
    // addresses) is paid by half the threads (2325 bfloat16 columns: 176 -> 159 us for 40 001 rows)
    s.units = units <= 128 ? 1 : units <= 1024 ? 2 : 4;
    if (units <= 2048) s.threads = (int)((units + s.units * 32 - 1) / (s.units * 32) * 32);
    const int64_t resident =
        s.threads ? std::max<int64_t>(1, std::min<int64_t>((s.units == 1 ? 1024 : 512) / s.threads, 16)) : 8;
    // a multiple of eight, so that the rows of one CTA are aligned alike; or a CTA a row
    s.grid = std::max<int64_t>(1, std::min<int64_t>(rows, std::max<int64_t>(8, resident * sms / 8 * 8)));
    s.bytes = (size_t)s.grid * s.pitch * sizeof(float) + (s.threads ? 0 : (size_t)rows * sizeof(float));
    return s;
}

// Whether rows of a matrix sit like those of `s` relative to 16 bytes.
template <class T>
bool alike(const T* p, int64_t stride, const MatrixIn<T>& s) {
    return reinterpret_cast<uintptr_t>(p) % 16 == reinterpret_cast<uintptr_t>(s.data) % 16 &&
           (stride - s.stride) * (int64_t)sizeof(T) % 16 == 0;
}

template <class T>
void norm_backward(NormBackwardArgs<T> a, float* dweight, const BackwardShape& s, int device, cudaStream_t stream) {
    if (s.threads) {
        const bool same = alike(a.dy.data, a.dy.stride, a.s) && alike(static_cast<const T*>(a.dx), a.dx_stride, a.s) &&
                          (!a.dsum || alike(a.dsum, a.dsum_stride, a.s));
        const auto kernel = s.units == 1   ? (same ? norm_backward_kernel<T, 1, true> : norm_backward_kernel<T, 1, false>)
                            : s.units == 2 ? (same ? norm_backward_kernel<T, 2, true> : norm_backward_kernel<T, 2, false>)
                                           : (same ? norm_backward_kernel<T, 4, true> : norm_backward_kernel<T, 4, false>);
        const int bytes_a_thread = ring_depth(s.units) * 3 * s.units * 16, bytes = bytes_a_thread * s.threads;  // at most 192 KB
        // raised once to what the widest CTA of this kernel takes: other calls may launch it with other widths meanwhile
        static std::atomic<uint64_t> done[3][2];
        allow_shared(kernel, bytes_a_thread * 512, done[s.units / 2][same], device, "norm gradient ring");
        kernel<<<(unsigned)s.grid, s.threads, bytes, stream>>>(a);
    } else {
        a.dots = a.partial + s.grid * s.pitch;
        norm_dots_kernel<T><<<(unsigned)a.s.rows, 256, 0, stream>>>(a);
        check(cudaGetLastError(), "norm gradient launch");
        const int64_t stripes = (a.s.width + 256 * kUnit<T> - 1) / (256 * kUnit<T>);
        need(stripes <= 65535, "readout: norm gradient too wide");
        norm_stripes_kernel<T><<<dim3((unsigned)s.grid, (unsigned)stripes), 256, 0, stream>>>(a);
    }
    check(cudaGetLastError(), "norm gradient launch");
    column_sum_kernel<<<(unsigned)((a.s.width + 31) / 32), 1024, 0, stream>>>(a.partial, s.pitch, (int)s.grid, a.s.width,
                                                                            dweight);
    check(cudaGetLastError(), "norm gradient launch");
}

// ------------------------------------------------------------ block quantiser

template <class T>
struct TileArgs {
    MatrixIn<T> x;
    const float* row_factor;
    const float* col_factor;
    uint8_t* codes;  // [rows][code_stride]
    int64_t code_stride;
    float* scales;
    int64_t scale_stride;
    uint8_t* codes_t;  // [width][code_t_stride]
    int64_t code_t_stride;
    float* scales_t;
    int64_t scale_t_stride;
};

// One CTA a tile of 128 rows x 128 columns, read once into registers: warp w
// holds rows 16 w .. 16 w + 15, a lane four neighbouring columns of each.
// Blocks along the rows are reduced inside the warp, blocks along the columns
// over the warps through shared memory.  The transposed codes meet in a 16 KB
// tile of shared memory whose 16-byte pieces (16 rows of a column) are placed at
// piece ^ column / 4, so that both the stores of a lane's four columns and the
// reads along a column are free of bank conflicts.
// TILES: one scale for the whole tile, in both directions.
// HBM would bound it (every element once in, one byte out a direction), but a
// tile's loads and its quantisations follow each other, and the registers leave
// too few warps (23 % both ways, 35 % along columns) to overlap those of other
// tiles: 65 536 x 3696 bfloat16 with row factors along columns 157 to 164 us by
// board, 4.5 to 4.7 TB/s, 56 % of issue slots used; 32 771 x 1024 both ways 39 us,
// 3.5 TB/s, 57 %.  Rows that are not aligned
// to words cost two reads and a splice a quad: 32 427 x 1857 both ways 96 us.  A persistent form that
// read the next tile ahead took 232 and 55 us: its addresses cost it registers.
//
// Two CTAs an SM with both directions of 16-bit elements (32 771 x 1024 on one
// board: 37 us, 45 with three, whose 80 registers do not hold the passes), else three, or two
// for the 64 registers that float32 quads fill.
template <class T, bool ROWS, bool TILES>
__global__ __launch_bounds__(256, sizeof(T) == 4 || (ROWS && !TILES) ? 2 : 3) void tile_kernel(const __grid_constant__ TileArgs<T> a) {
    using Word = typename Quad<T>::Word;
    __shared__ __align__(16) uint8_t s_codes[128 * 128];
    __shared__ __align__(16) float s_top[8][128];
    __shared__ __align__(16) float s_factor[128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t tile_row = (int64_t)blockIdx.y * 128, tile_col = (int64_t)blockIdx.x * 128;
    const int row0 = warp * 16, col0 = lane * 4;
    const int64_t rows = a.x.rows, width = a.x.width, col = tile_col + col0;
    const uintptr_t begin = reinterpret_cast<uintptr_t>(a.x.data);
    const uintptr_t end = reinterpret_cast<uintptr_t>(a.x.data + (rows - 1) * a.x.stride + width);

    Word raw[16];
    const T* from = a.x.data + (tile_row + row0) * a.x.stride;
    if (tile_row + 128 <= rows && tile_col + 128 <= width && quads_aligned(a.x.data) &&
        a.x.stride * sizeof(T) % sizeof(Word) == 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) raw[i] = __ldg(reinterpret_cast<const Word*>(from + i * a.x.stride + col));
    } else if (tile_row + 128 < rows && (tile_row > 0 || tile_col > 0)) {
        // words of any alignment: something of the matrix lies before and after this tile's part of every row
        if (col + 4 <= width) {
#pragma unroll
            for (int i = 0; i < 16; ++i) raw[i] = load_split(from + i * a.x.stride + col);
        } else {  // the row ends in or before the quad
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                raw[i] = Word{};
                T* t = reinterpret_cast<T*>(&raw[i]);
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (col + e < width) t[e] = from[i * a.x.stride + col + e];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            raw[i] = tile_row + row0 + i < rows ? load_quad(from + i * a.x.stride, col, width, begin, end) : Word{};
    }
    // along a column its own factor cancels, only the rows' factors enter the codes, and the other way round
    const bool row_factor = !TILES && a.row_factor, col_factor = ROWS && !TILES && a.col_factor;
    if (row_factor) {
        if (threadIdx.x < 128)
            s_factor[threadIdx.x] = tile_row + threadIdx.x < rows ? a.row_factor[tile_row + threadIdx.x] : 0.0f;
        __syncthreads();
    }
    float g[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    if (col_factor) load_vector<4>(a.col_factor, col, width, g);

    float4 col_top = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        float4 x = unpack4<T>(raw[i]), y = unpack4<T>(raw[i + 1]);
        if (row_factor) {
            const float2 f = *reinterpret_cast<const float2*>(&s_factor[row0 + i]);
            x.x *= f.x, x.y *= f.x, x.z *= f.x, x.w *= f.x;
            y.x *= f.y, y.y *= f.y, y.z *= f.y, y.w *= f.y;
        }
        col_top = make_float4(larger(col_top.x, x.x, y.x), larger(col_top.y, x.y, y.y), larger(col_top.z, x.z, y.z),
                              larger(col_top.w, x.w, y.w));
    }
    // Between the passes over the quads: they are unpacked again each time, 64 floats would not fit the registers.
    const auto forget = [&] {
#pragma unroll
        for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(raw[i].x), "+r"(raw[i].y));
    };
    forget();
    if constexpr (ROWS && !TILES) {
        // The rows' maxima first; lane i then works out row i's factor for all lanes.
        float mine = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float4 x = unpack4<T>(raw[i]);
            if (col_factor) x.x *= g[0], x.y *= g[1], x.z *= g[2], x.w *= g[3];
            const float top = warp_larger(larger(larger(x.x, x.y, x.z), x.w));
            if (lane == i) mine = top;
        }
        const Factor own(mine);
        forget();
        const int64_t own_row = tile_row + row0 + lane;
        if (lane < 16 && own_row < rows)
            a.scales[own_row * a.scale_stride + blockIdx.x] = scale_of(mine) * (row_factor ? s_factor[row0 + lane] : 1.0f);
        uint8_t* out = a.codes + (tile_row + row0) * a.code_stride + col;
        const int here = col < width ? (int)min((int64_t)16, rows - tile_row - row0) : 0;  // rows to write
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float4 x = unpack4<T>(raw[i]);
            Factor factor(0.0f);
            factor.inverse = __shfl_sync(0xffffffffu, own.inverse, i);
            factor.scale = __shfl_sync(0xffffffffu, own.scale, i);
            uint32_t q;
            if (col_factor) {
                q = codes4(factor(x.x * g[0]), factor(x.y * g[1]), factor(x.z * g[2]), factor(x.w * g[3]));
            } else {
                q = codes4(factor(x.x), factor(x.y), factor(x.z), factor(x.w));
            }
            if (i < here) *reinterpret_cast<uint32_t*>(out) = q;
            out += a.code_stride;
            asm volatile("" : "+l"(out));  // one address on its way through the rows, not sixteen
        }
        forget();
    }

    if constexpr (TILES) {
        const float mine = warp_larger(larger(larger(larger(col_top.x, col_top.y), col_top.z), col_top.w));
        if (lane == 0) s_top[0][warp] = mine;
        __syncthreads();
        float top = s_top[0][0];
#pragma unroll
        for (int w = 1; w < 8; ++w) top = larger(top, s_top[0][w]);
        col_top = make_float4(top, top, top, top);
        if (threadIdx.x == 0) {
            if constexpr (ROWS) a.scales[blockIdx.y * a.scale_stride + blockIdx.x] = scale_of(top);
            a.scales_t[blockIdx.x * a.scale_t_stride + blockIdx.y] = scale_of(top);
        }
    } else {
        *reinterpret_cast<float4*>(&s_top[warp][col0]) = col_top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const float4 other = *reinterpret_cast<const float4*>(&s_top[w][col0]);
            col_top = make_float4(larger(col_top.x, other.x), larger(col_top.y, other.y), larger(col_top.z, other.z),
                                  larger(col_top.w, other.w));
        }
        if (warp == 0) {
            const float top[4] = {col_top.x, col_top.y, col_top.z, col_top.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < width)
                    a.scales_t[(col + j) * a.scale_t_stride + blockIdx.y] =
                        scale_of(top[j]) * (a.col_factor ? a.col_factor[col + j] : 1.0f);
        }
    }

#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const Factor factor(j == 0 ? col_top.x : j == 1 ? col_top.y : j == 2 ? col_top.z : col_top.w);
        const auto entry = [&](int i) { return to_float(reinterpret_cast<const T*>(&raw[i])[j]); };
        uint32_t piece[4];
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            if (row_factor) {
                const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(&s_factor[row0 + i]);
                float q[4];
                factor.pair(entry(i), entry(i + 1), f.x, q[0], q[1]);
                factor.pair(entry(i + 2), entry(i + 3), f.y, q[2], q[3]);
                piece[i / 4] = codes4(q[0], q[1], q[2], q[3]);
            } else {
                piece[i / 4] = codes4(factor(entry(i)), factor(entry(i + 1)), factor(entry(i + 2)), factor(entry(i + 3)));
            }
        }
        *reinterpret_cast<uint4*>(s_codes + (col0 + j) * 128 + (warp ^ (lane & 7)) * 16) =
            make_uint4(piece[0], piece[1], piece[2], piece[3]);
    }
    if constexpr (TILES && ROWS) {
        forget();
        const Factor factor(col_top.x);
        uint8_t* out = a.codes + (tile_row + row0) * a.code_stride + col;
        const int here = col < width ? (int)min((int64_t)16, rows - tile_row - row0) : 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float4 x = unpack4<T>(raw[i]);
            if (i < here)
                *reinterpret_cast<uint32_t*>(out) = codes4(factor(x.x), factor(x.y), factor(x.z), factor(x.w));
            out += a.code_stride;
            asm volatile("" : "+l"(out));
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int at = k * 256 + threadIdx.x;
        const int c = at >> 3, piece = at & 7;
        const uint4 v = *reinterpret_cast<const uint4*>(s_codes + c * 128 + (piece ^ (c / 4 & 7)) * 16);
        const int64_t row = tile_row + piece * 16;
        if (tile_col + c < width && row < rows)  // the pitch covers the 16 bytes
            *reinterpret_cast<uint4*>(a.codes_t + (tile_col + c) * a.code_t_stride + row) = v;
    }
}

template <class T, bool ROWS, bool TILES>
void launch_tiles(const TileArgs<T>& a, cudaStream_t stream) {
    const int64_t cols = blocks_of(a.x.width), rows = blocks_of(a.x.rows);
    if (cols == 0 || rows == 0) return;
    if (cols > 0x7fffffff) raise(MDSOAP_INVALID_ARGUMENT, "quantize: matrix too wide");
    // grid.y holds 65 535 tiles: taller matrices go in slabs of rows
    for (int64_t r0 = 0; r0 < rows; r0 += 65535) {
        TileArgs<T> b = a;
        const int64_t count = std::min<int64_t>(65535, rows - r0), skip = r0 * 128;
        b.x.data += skip * a.x.stride;
        b.x.rows = std::min<int64_t>(a.x.rows - skip, count * 128);
        if (b.row_factor) b.row_factor += skip;
        if (b.codes) b.codes += skip * a.code_stride;
        if (b.scales) b.scales += (TILES ? r0 : skip) * a.scale_stride;
        if (b.codes_t) b.codes_t += skip;
        if (b.scales_t) b.scales_t += r0;
        tile_kernel<T, ROWS, TILES><<<dim3((unsigned)cols, (unsigned)count), 256, 0, stream>>>(b);
        check(cudaGetLastError(), "quantize launch");
    }
}

// ------------------------------------------------------------ argument checks

void check_matrix(const void* data, int64_t rows, int64_t width, int64_t stride, const char* what) {
    const bool ok = rows >= 0 && width >= 0 && (rows <= 1 || stride >= width) && (rows == 0 || width == 0 || data);
    if (!ok) raise(MDSOAP_INVALID_ARGUMENT, std::string("readout: invalid ") + what);
}

// The row kernel counts columns in 32 bits, past a row's end too.
constexpr int64_t kWidest = int64_t(1) << 30;

void check_codes(const void* codes, int64_t rows, int64_t width, int64_t stride, const void* scales,
                 int64_t scale_rows, int64_t scale_stride, const char* what) {
    const bool empty = rows == 0 || width == 0;
    const bool ok = empty || (codes && scales && reinterpret_cast<uintptr_t>(codes) % 16 == 0 && stride % 16 == 0 &&
                              stride >= width && (scale_rows <= 1 || scale_stride >= blocks_of(width)));
    if (!ok)
        raise(MDSOAP_INVALID_ARGUMENT,
              std::string("readout: ") + what + " need a 16-byte aligned base, a pitch that is a multiple of 16 and "
                                                "one scale for each block of 128");
}

}  // namespace

extern "C" {

int mdsoap_rms_norm(const void* x, int64_t rows, int64_t width, int64_t x_stride, const void* residual,
                    int64_t residual_stride, int32_t dtype, const float* weight, double eps, void* sum,
                    int64_t sum_stride, float* rstd, void* out, int64_t out_stride, float* scales, int64_t scale_stride,
                    int32_t device, void* stream) {
    return entry([&] {
        check_matrix(x, rows, width, x_stride, "norm input");
        check_matrix(residual ? residual : x, rows, width, residual ? residual_stride : x_stride, "norm residual");
        need(width <= kWidest, "readout: norm input wider than 2^30 columns");
        need(weight || width == 0, "readout: the norm needs a weight");
        // the kernel holds it in float32, where a smaller one is zero: a row of zeros would get an infinite factor
        need((float)eps > 0.0f && eps < 1e30, "readout: eps must be positive (in float32, too)");
        if (sum) check_matrix(sum, rows, width, sum_stride, "norm sum");
        if (scales) check_codes(out, rows, width, out_stride, scales, rows, scale_stride, "8-bit rows");
        else check_matrix(out, rows, width, out_stride, "norm output");
        const OnDevice current(device);
        if (width == 0 && rows > 0 && rstd)  // the mean of no entries: NaN, here from bytes of all ones
            check(cudaMemsetAsync(rstd, 0xff, rows * sizeof(float), static_cast<cudaStream_t>(stream)), "norm of no columns");
        by_type(dtype, [&](auto tag) {
            using T = decltype(tag);
            RowArgs<T> a{};
            a.x = {static_cast<const T*>(x), rows, width, x_stride};
            a.residual = static_cast<const T*>(residual);
            a.residual_stride = residual_stride;
            a.col_factor = weight;
            a.eps = (float)eps;
            a.sum = static_cast<T*>(sum);
            a.sum_stride = sum_stride;
            a.rstd = rstd;
            if (scales) {
                a.codes = static_cast<uint8_t*>(out);
                a.code_stride = out_stride;
                a.scales = scales;
                a.scale_stride = scale_stride;
                launch_rows<T, Rows::Norm8>(a, device, static_cast<cudaStream_t>(stream));
            } else {
                a.wide = static_cast<T*>(out);
                a.wide_stride = out_stride;
                launch_rows<T, Rows::NormWide>(a, device, static_cast<cudaStream_t>(stream));
            }
        });
    });
}

int mdsoap_rms_norm_backward_bytes(int64_t rows, int64_t width, int32_t dtype, int32_t device, int64_t* bytes) {
    return entry([&] {
        need(rows >= 0 && width >= 0 && bytes, "readout: invalid norm gradient shape");
        by_type(dtype, [&](auto tag) {
            *bytes = (int64_t)backward_shape(rows, width, kUnit<decltype(tag)>, sm_count(device)).bytes;
        });
    });
}

int mdsoap_rms_norm_backward(const void* dy, int64_t rows, int64_t width, int64_t dy_stride, const void* sum,
                             int64_t sum_stride, const float* rstd, const float* weight, const void* dsum,
                             int64_t dsum_stride, int32_t dtype, void* dx, int64_t dx_stride, float* dweight,
                             void* workspace, int64_t workspace_bytes, int32_t device, void* stream) {
    return entry([&] {
        check_matrix(dy, rows, width, dy_stride, "norm gradient dy");
        check_matrix(sum, rows, width, sum_stride, "norm gradient sum");
        check_matrix(dx, rows, width, dx_stride, "norm gradient dx");
        if (dsum) check_matrix(dsum, rows, width, dsum_stride, "norm gradient dsum");
        need(rows <= 0x7fffffff, "readout: too many rows");
        need(width == 0 || (weight && dweight), "readout: the norm gradient needs weight and dweight");
        need(rows == 0 || width == 0 || rstd, "readout: the norm gradient needs rstd");
        if (width == 0) return;
        const OnDevice current(device);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (rows == 0) {
            check(cudaMemsetAsync(dweight, 0, width * sizeof(float), s), "clear weight gradient");
            return;
        }
        by_type(dtype, [&](auto tag) {
            using T = decltype(tag);
            const BackwardShape shape = backward_shape(rows, width, kUnit<T>, sm_count(device));
            need(workspace && workspace_bytes >= (int64_t)shape.bytes &&
                     reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                 "readout: norm gradient workspace too small or not 16-byte aligned");
            NormBackwardArgs<T> a{};
            a.dy = {static_cast<const T*>(dy), rows, width, dy_stride};
            a.s = {static_cast<const T*>(sum), rows, width, sum_stride};
            a.dsum = static_cast<const T*>(dsum);
            a.dsum_stride = dsum_stride;
            a.rstd = rstd;
            a.weight = weight;
            a.dx = static_cast<T*>(dx);
            a.dx_stride = dx_stride;
            a.partial = static_cast<float*>(workspace);
            a.pitch = shape.pitch;
            norm_backward<T>(a, dweight, shape, device, s);
        });
    });
}

int mdsoap_quantize(const void* x, int64_t rows, int64_t width, int64_t x_stride, int32_t dtype,
                    const float* row_factor, const float* col_factor, int32_t tiles, void* codes, int64_t code_stride,
                    float* scales, int64_t scale_stride, void* codes_t, int64_t code_t_stride, float* scales_t,
                    int64_t scale_t_stride, int32_t device, void* stream) {
    return entry([&] {
        check_matrix(x, rows, width, x_stride, "matrix to quantize");
        need(codes || codes_t, "readout: quantize needs an output");
        need(!tiles || (!row_factor && !col_factor), "readout: tiles take no factors");
        need(!tiles || codes_t, "readout: tiles come with their transpose");
        if (codes)
            check_codes(codes, rows, width, code_stride, scales, tiles ? blocks_of(rows) : rows, scale_stride,
                        "8-bit rows");
        if (codes_t)
            check_codes(codes_t, width, rows, code_t_stride, scales_t, tiles ? blocks_of(width) : width,
                        scale_t_stride, "8-bit columns");
        const OnDevice current(device);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        by_type(dtype, [&](auto tag) {
            using T = decltype(tag);
            if (codes && !codes_t) {
                RowArgs<T> a{};
                a.x = {static_cast<const T*>(x), rows, width, x_stride};
                a.col_factor = col_factor;
                a.row_factor = row_factor;
                a.codes = static_cast<uint8_t*>(codes);
                a.code_stride = code_stride;
                a.scales = scales;
                a.scale_stride = scale_stride;
                launch_rows<T, Rows::Quantize>(a, device, s);
                return;
            }
            const TileArgs<T> a{{static_cast<const T*>(x), rows, width, x_stride},
                                row_factor, col_factor,
                                static_cast<uint8_t*>(codes), code_stride, scales, scale_stride,
                                static_cast<uint8_t*>(codes_t), code_t_stride, scales_t, scale_t_stride};
            if (tiles && codes) launch_tiles<T, true, true>(a, s);
            else if (tiles) launch_tiles<T, false, true>(a, s);
            else if (codes) launch_tiles<T, true, false>(a, s);
            else launch_tiles<T, false, false>(a, s);
        });
    });
}

}  // extern "C"
