// Readout operators on rows: root-mean-square norm with the residual's
// addition (wide or 8-bit output), its gradient, and the 8-bit block
// quantiser, with their C entry points (include/mdsoap.h).
#include "host_errors.cuh"
#include "readout.cuh"
#include "readout_host.cuh"

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

// One row by one warp (CTA_ROW false) or by the CTA's warps together.
//
// s = x + r; rstd = (mean s^2 + eps)^-1/2; y = s rstd w.  In 8 bits the factor
// rstd is constant in the row, so it cancels from the codes 448 z / max|z| of
// z = s w and lives in the scales alone: the codes are written in the one pass
// that also sums s^2, and only the blocks' maxima wait for the row's end (in
// shared memory, one float a block).  Nothing of the row is held or read twice.
// Bound by HBM: x and r once in, sum and codes once out.
template <class T, bool CTA_ROW, Rows MODE>
__global__ __launch_bounds__(kRowWarps * 32) void rows_kernel(const __grid_constant__ RowArgs<T> a) {
    constexpr int N = kUnit<T>;
    constexpr int kChunk = 32 * N;            // columns a warp takes at a time
    constexpr int kLanes = kBlock / N;        // lanes of one block of 128: 16 or 32
    extern __shared__ float s_top[];
    __shared__ float s_sum[kRowWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = CTA_ROW ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kRowWarps + warp;
    if (row >= a.x.rows) return;  // never with CTA_ROW, whose warps meet below
    const int64_t width = a.x.width;
    const int64_t nblocks = (width + kBlock - 1) / kBlock;
    float* const top = s_top + (CTA_ROW ? 0 : warp * nblocks);
    const MatrixIn<T> r{a.residual, a.x.rows, width, a.residual_stride};
    const int64_t step = (CTA_ROW ? kRowWarps : 1) * (int64_t)kChunk;
    const int64_t first = (CTA_ROW ? warp * (int64_t)kChunk : 0) + lane * N;

    float total = 0.0f;
    for (int64_t col = first; col - lane * N < width; col += step) {
        float s[N];
        unpack<T>(a.x.unit(row, col), s);
        if (a.residual) {
            float f[N];
            unpack<T>(r.unit(row, col), f);
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] += f[i];
        }
        if constexpr (MODE != Rows::Quantize) {
#pragma unroll
            for (int i = 0; i < N; ++i) total = fmaf(s[i], s[i], total);
            if (a.sum) store_unit(a.sum + row * a.sum_stride, col, width, pack<T>(s));
        }
        if constexpr (MODE != Rows::NormWide) {
            if (a.col_factor) {
                float w[N];
                load_vector<N>(a.col_factor, col, width, w);
#pragma unroll
                for (int i = 0; i < N; ++i) s[i] *= w[i];
            }
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) most = max(most, magnitude(s[i]));
#pragma unroll
            for (int d = kLanes / 2; d; d >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
            const float block_top = __uint_as_float(most);
            if (col < width) {
                if (lane % kLanes == 0) top[col / kBlock] = block_top;
                const Factor factor(block_top);
                uint8_t* out = a.codes + row * a.code_stride + col;  // the pitch covers the unit's padding
                if constexpr (N == 8) {
                    *reinterpret_cast<uint2*>(out) =
                        make_uint2(codes4(factor(s[0]), factor(s[1]), factor(s[2]), factor(s[3])),
                                   codes4(factor(s[4]), factor(s[5]), factor(s[6]), factor(s[7])));
                } else {
                    *reinterpret_cast<uint32_t*>(out) = codes4(factor(s[0]), factor(s[1]), factor(s[2]), factor(s[3]));
                }
            }
        }
    }

    float row_scale = 1.0f;
    if constexpr (MODE != Rows::Quantize) {
        total = warp_sum(total);
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
        row_scale = a.row_factor[row];
    }
    if constexpr (CTA_ROW) __syncthreads();
    __syncwarp();

    if constexpr (MODE == Rows::NormWide) {
        for (int64_t col = first; col - lane * N < width; col += step) {
            float s[N], w[N];
            unpack<T>(a.x.unit(row, col), s);
            if (a.residual) {
                float f[N];
                unpack<T>(r.unit(row, col), f);
#pragma unroll
                for (int i = 0; i < N; ++i) s[i] += f[i];
            }
            load_vector<N>(a.col_factor, col, width, w);
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] = s[i] * row_scale * w[i];
            store_unit(a.wide + row * a.wide_stride, col, width, pack<T>(s));
        }
    } else {
        // A negative row factor turns the signs of the codes, which are written
        // already: the quantiser takes it through its scale's sign instead.
        const int at = CTA_ROW ? threadIdx.x : lane;
        for (int64_t b = at; b < nblocks; b += CTA_ROW ? kRowWarps * 32 : 32)
            a.scales[row * a.scale_stride + b] = scale_of(top[b]) * row_scale;
    }
}

template <class T, Rows MODE>
void launch_rows(const RowArgs<T>& a, int sms, cudaStream_t stream) {
    if (a.x.rows == 0 || a.x.width == 0) return;
    const int64_t nblocks = blocks_of(a.x.width);
    const bool tops = MODE != Rows::NormWide;
    const size_t warp_bytes = tops ? nblocks * sizeof(float) : 0;
    if (warp_bytes > 200 * 1024) raise(MDSOAP_INVALID_ARGUMENT, "readout rows: width exceeds 6 553 600 columns");
    // A warp a row keeps all reductions inside the warp; a CTA a row when there
    // are too few rows to fill the SMs that way, or the maxima of eight rows
    // would not fit.
    const bool cta_row = a.x.rows < (int64_t)sms * kRowWarps * 2 || warp_bytes * kRowWarps > 48 * 1024;
    if (cta_row) {
        auto kernel = rows_kernel<T, true, MODE>;
        if (warp_bytes > 48 * 1024)
            check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)warp_bytes),
                  "readout rows: shared memory");
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
// A CTA of G threads takes rows b, b + grid, ...: each thread owns the same NU
// units of every row, so the row stays in registers between the sum c and the
// result, and the weight's gradient adds up in registers over the CTA's rows.
// The partial sums of all CTAs go to the workspace and are added in CTA order
// by a second kernel: the same bits on every run.  Bound by HBM: dy, s, dsum
// once in, ds once out.
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

template <int G>
__device__ __forceinline__ float cta_sum(float x, float* scratch) {
    x = warp_sum(x);
    if constexpr (G == 32) return x;
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < G / 32; ++w) total += scratch[w];
    return total;
}

template <class T, int G, int NU>
__global__ __launch_bounds__(G) void norm_backward_kernel(const __grid_constant__ NormBackwardArgs<T> a) {
    constexpr int N = kUnit<T>;
    __shared__ float scratch[2][G / 32];
    const int64_t width = a.s.width;
    const MatrixIn<T> dsum{a.dsum, a.s.rows, width, a.dsum_stride};
    float w[NU][N], dw[NU][N];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        load_vector<N>(a.weight, ((int64_t)u * G + threadIdx.x) * N, width, w[u]);
#pragma unroll
        for (int i = 0; i < N; ++i) dw[u][i] = 0.0f;
    }
    const float inv_width = __fdiv_rn(1.0f, (float)width);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.s.rows; row += gridDim.x, turn ^= 1) {
        uint4 qdy[NU], qs[NU], qd[NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int64_t col = ((int64_t)u * G + threadIdx.x) * N;
            qdy[u] = a.dy.unit(row, col);
            qs[u] = a.s.unit(row, col);
            if (a.dsum) qd[u] = dsum.unit(row, col);
        }
        const float rstd = a.rstd[row];
        float c = 0.0f;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            float dy[N], s[N];
            unpack<T>(qdy[u], dy);
            unpack<T>(qs[u], s);
#pragma unroll
            for (int i = 0; i < N; ++i) c = fmaf(dy[i] * w[u][i], s[i], c);
        }
        // two scratch rows in turn: a warp may be one row ahead of another, never two
        c = cta_sum<G>(c, scratch[turn]) * inv_width * rstd * rstd;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int64_t col = ((int64_t)u * G + threadIdx.x) * N;
            float dy[N], s[N], out[N];
            unpack<T>(qdy[u], dy);
            unpack<T>(qs[u], s);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float hat = s[i] * rstd;
                dw[u][i] = fmaf(dy[i], hat, dw[u][i]);
                out[i] = rstd * fmaf(-s[i], c, dy[i] * w[u][i]);
            }
            if (a.dsum) {
                float d[N];
                unpack<T>(qd[u], d);
#pragma unroll
                for (int i = 0; i < N; ++i) out[i] += d[i];
            }
            store_unit(a.dx + row * a.dx_stride, col, width, pack<T>(out));
        }
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int64_t col = ((int64_t)u * G + threadIdx.x) * N;
        if (col < width) {  // the pitch covers a whole unit
            float4* p = reinterpret_cast<float4*>(a.partial + blockIdx.x * a.pitch + col);
#pragma unroll
            for (int i = 0; i < N; i += 4) p[i / 4] = make_float4(dw[u][i], dw[u][i + 1], dw[u][i + 2], dw[u][i + 3]);
        }
    }
}

// Rows too wide for one CTA's registers: c of each row first ...
template <class T>
__global__ __launch_bounds__(256) void norm_dots_kernel(const __grid_constant__ NormBackwardArgs<T> a) {
    constexpr int N = kUnit<T>;
    __shared__ float scratch[8];
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
    c = cta_sum<256>(c, scratch);
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

// dweight[d] = the CTAs' partial sums in order: 8 threads a column take every
// eighth row of `partial` each and are added in order.
__global__ __launch_bounds__(256) void column_sum_kernel(const float* partial, int64_t pitch, int count, int64_t width,
                                                         float* out) {
    __shared__ float s[8][33];
    const int64_t col = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int part = threadIdx.x >> 5;
    float total = 0.0f;
    if (col < width) {
        int b = part;
        for (; b + 24 < count; b += 32) {
            const float v0 = partial[b * pitch + col], v1 = partial[(b + 8) * pitch + col],
                        v2 = partial[(b + 16) * pitch + col], v3 = partial[(b + 24) * pitch + col];
            total += (v0 + v1) + (v2 + v3);
        }
        for (; b < count; b += 8) total += partial[b * pitch + col];
    }
    s[part][threadIdx.x & 31] = total;
    __syncthreads();
    if (part == 0 && col < width) {
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) total += s[i][threadIdx.x & 31];
        out[col] = total;
    }
}

struct BackwardShape {
    int threads, units;  // 0 threads: the two-kernel form
    int64_t grid, pitch;
    size_t bytes;
};

// Threads and units so that a row fits a CTA's registers (units x 16 bytes a
// thread); grids of about 2048 threads an SM.
BackwardShape backward_shape(int64_t rows, int64_t width, int unit, int sms) {
    BackwardShape s{};
    s.pitch = (width + 7) / 8 * 8;
    const int64_t units = (width + unit - 1) / unit;
    if (units <= 32) s.threads = 32, s.units = 1;
    else if (units <= 64) s.threads = 64, s.units = 1;
    else if (units <= 128) s.threads = 128, s.units = 1;
    else if (units <= 256) s.threads = 128, s.units = 2;
    else if (units <= 512) s.threads = 256, s.units = 2;
    else if (units <= 1024) s.threads = 512, s.units = 2;
    else if (units <= 2048) s.threads = 512, s.units = 4;
    const int64_t resident = s.threads ? std::min(1024 / s.threads, 16) : 8;
    s.grid = std::max<int64_t>(1, std::min<int64_t>(rows, resident * sms));
    s.bytes = (size_t)s.grid * s.pitch * sizeof(float) + (s.threads ? 0 : (size_t)rows * sizeof(float));
    return s;
}

template <class T, int G, int NU>
void launch_backward(const NormBackwardArgs<T>& a, const BackwardShape& s, cudaStream_t stream) {
    norm_backward_kernel<T, G, NU><<<(unsigned)s.grid, G, 0, stream>>>(a);
}

template <class T>
void norm_backward(NormBackwardArgs<T> a, float* dweight, const BackwardShape& s, cudaStream_t stream) {
    const int key = s.threads * 8 + s.units;
    switch (key) {
        case 32 * 8 + 1: launch_backward<T, 32, 1>(a, s, stream); break;
        case 64 * 8 + 1: launch_backward<T, 64, 1>(a, s, stream); break;
        case 128 * 8 + 1: launch_backward<T, 128, 1>(a, s, stream); break;
        case 128 * 8 + 2: launch_backward<T, 128, 2>(a, s, stream); break;
        case 256 * 8 + 2: launch_backward<T, 256, 2>(a, s, stream); break;
        case 512 * 8 + 2: launch_backward<T, 512, 2>(a, s, stream); break;
        case 512 * 8 + 4: launch_backward<T, 512, 4>(a, s, stream); break;
        default: {
            a.dots = a.partial + s.grid * s.pitch;
            norm_dots_kernel<T><<<(unsigned)a.s.rows, 256, 0, stream>>>(a);
            check(cudaGetLastError(), "norm gradient launch");
            const int64_t stripes = (a.s.width + 256 * kUnit<T> - 1) / (256 * kUnit<T>);
            norm_stripes_kernel<T><<<dim3((unsigned)s.grid, (unsigned)stripes), 256, 0, stream>>>(a);
        }
    }
    check(cudaGetLastError(), "norm gradient launch");
    column_sum_kernel<<<(unsigned)((a.s.width + 31) / 32), 256, 0, stream>>>(a.partial, s.pitch, (int)s.grid, a.s.width,
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
// holds rows 16 w .. 16 w + 15, a lane kUnit neighbouring columns of each of
// its rows.  Blocks along the rows are reduced inside a (half) warp, blocks
// along the columns over the warps through shared memory.  The transposed
// codes meet in a 16 KB tile of shared memory whose 8-byte pieces are placed
// at piece ^ (column / unit), so that both the stores of consecutive rows and
// the 16-byte reads along them are free of bank conflicts.
// TILES: one scale for the whole tile, in both directions.
// Bound by HBM: every element once in, one byte out a direction.
template <class T, bool ROWS, bool COLS, bool TILES>
__global__ __launch_bounds__(256) void tile_kernel(const __grid_constant__ TileArgs<T> a) {
    constexpr int N = kUnit<T>;
    constexpr int kLanes = kBlock / N;          // lanes of one row of the tile: 16 or 32
    constexpr int kPart = 32 / kLanes;          // rows a warp reads at a time
    constexpr int kMine = 16 / kPart;           // rows of one lane, consecutive
    __shared__ __align__(16) uint8_t s_codes[COLS ? 128 * 128 : 16];
    __shared__ uint32_t s_top[8][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t tile_row = (int64_t)blockIdx.y * 128, tile_col = (int64_t)blockIdx.x * 128;
    const int row0 = warp * 16 + lane / kLanes * kMine;
    const int col0 = lane % kLanes * N;
    const int64_t rows = a.x.rows, width = a.x.width;

    uint4 raw[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        raw[i] = tile_row + row0 + i < rows ? a.x.unit(tile_row + row0 + i, tile_col + col0) : make_uint4(0, 0, 0, 0);

    float g[N];
    if (!TILES && ROWS && a.col_factor) load_vector<N>(a.col_factor, tile_col + col0, width, g);

    uint32_t col_top[N];
#pragma unroll
    for (int j = 0; j < N; ++j) col_top[j] = 0;
    uint32_t all_top = 0;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        float z[N];
        unpack<T>(raw[i], z);
        const int64_t row = tile_row + row0 + i;
        if constexpr (COLS && !TILES) {
            // along a column its own factor cancels: only the rows' factors enter the codes
            const float f = a.row_factor && row < rows ? a.row_factor[row] : 1.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) col_top[j] = max(col_top[j], magnitude(z[j] * f));
        }
        if constexpr (TILES) {
#pragma unroll
            for (int j = 0; j < N; ++j) all_top = max(all_top, magnitude(z[j]));
        }
        if constexpr (ROWS && !TILES) {
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (a.col_factor) z[j] *= g[j];
                most = max(most, magnitude(z[j]));
            }
#pragma unroll
            for (int d = kLanes / 2; d; d >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
            const float top = __uint_as_float(most);
            const Factor factor(top);
            if (row < rows && tile_col + col0 < width) {
                uint8_t* out = a.codes + row * a.code_stride + tile_col + col0;
                if constexpr (N == 8)
                    *reinterpret_cast<uint2*>(out) =
                        make_uint2(codes4(factor(z[0]), factor(z[1]), factor(z[2]), factor(z[3])),
                                   codes4(factor(z[4]), factor(z[5]), factor(z[6]), factor(z[7])));
                else
                    *reinterpret_cast<uint32_t*>(out) = codes4(factor(z[0]), factor(z[1]), factor(z[2]), factor(z[3]));
                if (lane % kLanes == 0)
                    a.scales[row * a.scale_stride + blockIdx.x] =
                        scale_of(top) * (a.row_factor ? a.row_factor[row] : 1.0f);
            }
        }
    }
    if constexpr (!COLS) return;

    Factor tile_factor(0.0f);
    if constexpr (TILES) {
#pragma unroll
        for (int d = 16; d; d >>= 1) all_top = max(all_top, __shfl_xor_sync(0xffffffffu, all_top, d));
        if (lane == 0) s_top[warp][0] = all_top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) all_top = max(all_top, s_top[w][0]);
        const float top = __uint_as_float(all_top);
        tile_factor = Factor(top);
        if (threadIdx.x == 0) {
            if constexpr (ROWS) a.scales[blockIdx.y * a.scale_stride + blockIdx.x] = scale_of(top);
            a.scales_t[blockIdx.x * a.scale_t_stride + blockIdx.y] = scale_of(top);
        }
    } else {
        if constexpr (kPart == 2) {
#pragma unroll
            for (int j = 0; j < N; ++j) col_top[j] = max(col_top[j], __shfl_xor_sync(0xffffffffu, col_top[j], 16));
        }
        if (lane < kLanes) {
#pragma unroll
            for (int j = 0; j < N; ++j) s_top[warp][col0 + j] = col_top[j];
        }
        __syncthreads();
        if (threadIdx.x < 128) {
            uint32_t most = 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) most = max(most, s_top[w][threadIdx.x]);
            s_top[0][threadIdx.x] = most;  // each thread writes only the column that it alone reads
            const int64_t col = tile_col + threadIdx.x;
            if (col < width)
                a.scales_t[col * a.scale_t_stride + blockIdx.y] =
                    scale_of(__uint_as_float(most)) * (a.col_factor ? a.col_factor[col] : 1.0f);
        }
        __syncthreads();
    }

#pragma unroll
    for (int j4 = 0; j4 < N; j4 += 4) {
        uint32_t piece[4][kMine / 4];
        Factor column[4] = {Factor(0.0f), Factor(0.0f), Factor(0.0f), Factor(0.0f)};
        if constexpr (!TILES) {
#pragma unroll
            for (int j = 0; j < 4; ++j) column[j] = Factor(__uint_as_float(s_top[0][col0 + j4 + j]));
        }
#pragma unroll
        for (int i4 = 0; i4 < kMine; i4 += 4) {
            float q[4][4];  // [row][column]
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float z[N];
                unpack<T>(raw[i4 + i], z);
                const int64_t row = tile_row + row0 + i4 + i;
                const float f = !TILES && a.row_factor && row < rows ? a.row_factor[row] : 1.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) q[i][j] = TILES ? tile_factor(z[j4 + j]) : column[j](z[j4 + j] * f);
                if constexpr (TILES && ROWS) {
                    if (row < rows && tile_col + col0 < width)
                        *reinterpret_cast<uint32_t*>(a.codes + row * a.code_stride + tile_col + col0 + j4) =
                            codes4(q[i][0], q[i][1], q[i][2], q[i][3]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) piece[j][i4 / 4] = codes4(q[0][j], q[1][j], q[2][j], q[3][j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = col0 + j4 + j;
#pragma unroll
            for (int k = 0; k < kMine / 8; ++k) {
                const int at = (row0 / 8 + k) ^ (col / N & 15);
                *reinterpret_cast<uint2*>(s_codes + col * 128 + at * 8) =
                    make_uint2(piece[j][2 * k], piece[j][2 * k + 1]);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int at = k * 256 + threadIdx.x;
        const int col = at >> 3, pair = at & 7;
        const int swap = col / N & 15;
        uint4 v = *reinterpret_cast<const uint4*>(s_codes + col * 128 + ((pair ^ (swap >> 1)) * 16));
        if (swap & 1) v = make_uint4(v.z, v.w, v.x, v.y);
        const int64_t row = tile_row + pair * 16;
        if (tile_col + col < width && row < rows)  // the pitch covers the 16 bytes
            *reinterpret_cast<uint4*>(a.codes_t + (tile_col + col) * a.code_t_stride + row) = v;
    }
}

template <class T, bool ROWS, bool COLS, bool TILES>
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
        tile_kernel<T, ROWS, COLS, TILES><<<dim3((unsigned)cols, (unsigned)count), 256, 0, stream>>>(b);
        check(cudaGetLastError(), "quantize launch");
    }
}

// ------------------------------------------------------------ argument checks

void check_matrix(const void* data, int64_t rows, int64_t width, int64_t stride, const char* what) {
    const bool ok = rows >= 0 && width >= 0 && (rows <= 1 || stride >= width) && (rows == 0 || width == 0 || data);
    if (!ok) raise(MDSOAP_INVALID_ARGUMENT, std::string("readout: invalid ") + what);
}

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
        need(weight || width == 0, "readout: the norm needs a weight");
        need(eps > 0.0 && eps < 1e30, "readout: eps must be positive");
        if (sum) check_matrix(sum, rows, width, sum_stride, "norm sum");
        if (scales) check_codes(out, rows, width, out_stride, scales, rows, scale_stride, "8-bit rows");
        else check_matrix(out, rows, width, out_stride, "norm output");
        check(cudaSetDevice(device), "cudaSetDevice");
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
            const int sms = sm_count(device);
            if (scales) {
                a.codes = static_cast<uint8_t*>(out);
                a.code_stride = out_stride;
                a.scales = scales;
                a.scale_stride = scale_stride;
                launch_rows<T, Rows::Norm8>(a, sms, static_cast<cudaStream_t>(stream));
            } else {
                a.wide = static_cast<T*>(out);
                a.wide_stride = out_stride;
                launch_rows<T, Rows::NormWide>(a, sms, static_cast<cudaStream_t>(stream));
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
        check(cudaSetDevice(device), "cudaSetDevice");
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
            norm_backward<T>(a, dweight, shape, s);
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
        check(cudaSetDevice(device), "cudaSetDevice");
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
                launch_rows<T, Rows::Quantize>(a, sm_count(device), s);
                return;
            }
            const TileArgs<T> a{{static_cast<const T*>(x), rows, width, x_stride},
                                row_factor, col_factor,
                                static_cast<uint8_t*>(codes), code_stride, scales, scale_stride,
                                static_cast<uint8_t*>(codes_t), code_t_stride, scales_t, scale_t_stride};
            if (tiles && codes) launch_tiles<T, true, true, true>(a, s);
            else if (tiles) launch_tiles<T, false, true, true>(a, s);
            else if (codes) launch_tiles<T, true, true, false>(a, s);
            else launch_tiles<T, false, true, false>(a, s);
        });
    });
}

}  // extern "C"
