// AdamW over many tensors in one launch, with states in 32 bits or in 8, and
// its C entry points (include/mdsoap.h).
#include "readout_host.cuh"

#include <algorithm>
#include <cmath>
#include <memory>
#include <mutex>
#include <vector>

using namespace mdsoap;
using namespace mdsoap::readout;

namespace {

constexpr int kThreads = 256;
constexpr int kSpan = 4;                         // elements of one thread's unit
constexpr int kTileUnits = 4;                    // units of a thread in one tile
constexpr int kTile = kThreads * kSpan * kTileUnits;  // 4096 elements, a multiple of the block of 128
constexpr int kGrads = 448;                      // gradient pointers handed over in one launch's parameters
constexpr int kFewGrads = 24;

struct Tensor {
    uint8_t *p, *m, *v;
    float *m_scale, *v_scale;
    int64_t count;
    int64_t first;  // position in the optimizer's own numbering of elements, a multiple of 128
    float decay;    // weight decay
    int32_t vector;  // p, m and v can be read in units of four
};

// One tile: addresses of its first element, and how many it has.
struct alignas(16) Tile {
    uint8_t *p, *m, *v;
    float *m_scale, *v_scale;
    int64_t first;   // its first element in the optimizer's numbering
    int64_t offset;  // its first element in the tensor
    int32_t tensor;
    int32_t count;
    float decay;
    int32_t vector;
};
constexpr int kTileWords = sizeof(Tile) / 4;

struct StepSettings {
    const Tile* tiles;
    int32_t tile_count;
    int32_t first_tensor;  // of this launch: grads[0] belongs to it
    float lr, beta1, beta2, rest1, rest2, eps, step_size, root2, grad_scale;
    uint32_t key;
};
// A launch's parameters are copied with it: few gradients take a short form.
template <int GRADS>
struct StepArgs : StepSettings {
    const void* grads[GRADS];
};

// Two 16-bit random numbers of an element: a counter mixed by two rounds of
// shift, exclusive or and multiplication with odd constants (the fractional
// parts of square roots of small primes).  `start`: what a quad's elements share.
__device__ __forceinline__ uint32_t noise_start(int64_t element, uint32_t key) {
    return (uint32_t)element ^ ((uint32_t)(element >> 32) * 0x3C6EF373u) ^ key;
}
__device__ __forceinline__ uint32_t noise(uint32_t start, int i) {
    uint32_t h = start ^ i;  // a quad's first element is a multiple of four
    h = (h ^ h >> 16) * 0xA54FF53Bu;
    h = (h ^ h >> 15) * 0x510E527Fu;
    return h ^ h >> 16;
}

template <class T>
__device__ __forceinline__ void load4(const T* p, int at, int count, bool vector, float (&f)[4]) {
    if (vector && at + 4 <= count) {
        if constexpr (sizeof(T) == 4) {
            const float4 q = *reinterpret_cast<const float4*>(p + at);
            f[0] = q.x, f[1] = q.y, f[2] = q.z, f[3] = q.w;
        } else {
            const uint2 q = *reinterpret_cast<const uint2*>(p + at);
            const T* t = reinterpret_cast<const T*>(&q);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = to_float(t[i]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = at + i < count ? to_float(p[at + i]) : 0.0f;
}

template <class T>
__device__ __forceinline__ void store4(T* p, int at, int count, bool vector, const float (&f)[4]) {
    if (vector && at + 4 <= count) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p + at) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
            uint2 q;
            T* t = reinterpret_cast<T*>(&q);
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = from_float<T>(f[i]);
            *reinterpret_cast<uint2*>(p + at) = q;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i < count) p[at + i] = from_float<T>(f[i]);
}

__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, int at, int count, bool vector) {
    if (vector && at + 4 <= count) return *reinterpret_cast<const uint32_t*>(p + at);
    uint32_t q = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i < count) q |= (uint32_t)p[at + i] << (8 * i);
    return q;
}

__device__ __forceinline__ void store_codes(uint8_t* p, int at, int count, bool vector, uint32_t codes) {
    if (vector && at + 4 <= count) {
        *reinterpret_cast<uint32_t*>(p + at) = codes;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i < count) p[at + i] = (uint8_t)(codes >> (8 * i));
}

__device__ __forceinline__ void decode(uint32_t codes, float scale, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * i)), __NV_E4M3);
        const float2 t = __half22float2(__half2(h));
        f[2 * i] = t.x * scale, f[2 * i + 1] = t.y * scale;
    }
}

// The quick root, of every float32 size: a gradient's square leaves the normal
// range at both ends long before the gradient does.  (With v times 2^24,
// above the size where the quickest root counts as zero, a step of 8-bit states
// took 205 us in place of 209, but that is infinite from a v of 2^104 on.)
__device__ __forceinline__ float square_root(float x) {
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Codes of four values of the warp's block of 128, and the block's scale.
// a = |x| / scale (at most 448) goes down to an e4m3 value after u / 2^16 of
// that value's step has been added; `u20` holds the u, times 16.  From 2^-6 on
// the step is bit 20 of the float, so the sum's top bits are the code; below it
// is 2^-9 (rare: the warp looks whether it has such values at all).  The
// quotient is x times the approximate reciprocal with one correction by the
// exact remainder, which leaves the correctly rounded one but for about one in a
// million.  FLOOR: a positive x keeps at least the smallest code.
template <bool FLOOR>
__device__ __forceinline__ uint32_t encode(const float (&x)[4], const uint32_t (&u20)[4], float& scale) {
    const float top = warp_larger(larger(larger(x[0], x[1], x[2]), x[3]));
    scale = scale_of(top);
    const float inverse = reciprocal(scale);
    float a[4], least = kTop;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = fabsf(x[i]) * inverse;
        a[i] = fmaf(fmaf(-q, scale, fabsf(x[i])), inverse, q);
        least = fminf(least, a[i]);
    }
    uint32_t code[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) code[i] = (__float_as_uint(a[i]) + u20[i] - (960u << 20)) >> 20;
    if (__any_sync(0xffffffffu, least < 0x1p-6f)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float u = __uint_as_float(0x3f800000u | u20[i] << 3) - 1.0f;
            const float t = __fadd_rd(fmaf(a[i], 512.0f, u), 0x1p23f);  // floor into the low bits
            if (a[i] < 0x1p-6f) code[i] = __float_as_uint(t) & 15u;
            if (FLOOR && code[i] == 0 && x[i] > 0.0f) code[i] = 1;
        }
    }
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t c = min(code[i], 0x7eu);
        if (!FLOOR) c |= __float_as_uint(x[i]) >> 24 & 0x80u;
        codes |= c << (8 * i);
    }
    return scale == 0.0f ? 0u : codes;
}

// One CTA a tile of 4096 elements of one tensor.
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in float32, each stored value rounded once; root and quotient of p's update are
// the quick ones (2^-22 of the update).
// 8-bit states are e4m3 codes with a float32 scale for each block of 128
// elements of the tensor; a warp holds exactly one block at a time.  They are
// rounded by dithering: b2 = 0.999 moves v by a thousandth a step and the codes
// lie 1/16 to 1/8 apart, so to the nearest code v would stay where it is.  v
// itself is stored and not its root, whose dithering noise squared would add
// to v more than b2 takes away; a positive v keeps at least the smallest code,
// since a zero under a non-zero m would make a huge step.  A NaN or infinite
// moment shows in its block's scale.
// With 8-bit states neither HBM nor the arithmetic is full: 64 M elements in 211
// tensors, float32 p, bfloat16 g, 209 us a step (204 to 212 by board), 4.3 TB/s,
// 70 % of issue slots used by a third of the warps that fit (365 us with exact
// divisions and codes by conversion).
template <class P, class G, bool SMALL>
struct Update {
    const StepSettings& a;
    const Tile& t;
    const G* g;
    float keep;

    struct Unit {
        float x[4], y[4], m[4], v[4];
        uint32_t qm, qv;
        float sm, sv;
    };

    // `at`: the lane's first element in the tile, a multiple of four.
    __device__ __forceinline__ void load(Unit& u, int at, int count, bool vec_p, bool vec_g) const {
        load4(reinterpret_cast<const P*>(t.p), at, count, vec_p, u.x);
        load4(g, at, count, vec_g, u.y);
        if constexpr (SMALL) {
            u.qm = load_codes(t.m, at, count, vec_p);
            u.qv = load_codes(t.v, at, count, vec_p);
            u.sm = t.m_scale[at / kBlock], u.sv = t.v_scale[at / kBlock];  // the warp's first lane has an element of it
        } else {
            load4(reinterpret_cast<const float*>(t.m), at, count, vec_p, u.m);
            load4(reinterpret_cast<const float*>(t.v), at, count, vec_p, u.v);
        }
    }

    __device__ __forceinline__ void finish(Unit& u, int at, int count, bool vec_p) const {
        if constexpr (SMALL) {
            decode(u.qm, u.sm, u.m);
            decode(u.qv, u.sv, u.v);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float grad = u.y[i] * a.grad_scale;
            // products rounded, then the sum: the states' codes depend on every bit of it
            u.m[i] = __fadd_rn(__fmul_rn(a.beta1, u.m[i]), __fmul_rn(a.rest1, grad));
            u.v[i] = __fadd_rn(__fmul_rn(a.beta2, u.v[i]), __fmul_rn(__fmul_rn(a.rest2, grad), grad));
            const float root = fmaf(square_root(u.v[i]), a.root2, a.eps);
            u.x[i] = fmaf(-a.step_size, u.m[i] * reciprocal(root), u.x[i] * keep);
        }
        store4(reinterpret_cast<P*>(t.p), at, count, vec_p, u.x);
        if constexpr (SMALL) {
            const uint32_t start = noise_start(t.first + at, a.key);
            uint32_t um[4], uv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t h = noise(start, i);
                um[i] = h >> 12 & 0xffff0u, uv[i] = h << 4 & 0xffff0u;
            }
            float sm, sv;
            store_codes(t.m, at, count, vec_p, encode<false>(u.m, um, sm));
            store_codes(t.v, at, count, vec_p, encode<true>(u.v, uv, sv));
            if ((threadIdx.x & 31) == 0) t.m_scale[at / kBlock] = sm, t.v_scale[at / kBlock] = sv;
        } else {
            store4(reinterpret_cast<float*>(t.m), at, count, vec_p, u.m);
            store4(reinterpret_cast<float*>(t.v), at, count, vec_p, u.v);
        }
    }
};

// Persistent: a CTA takes tiles b, b + grid, ...; records are read two tiles
// ahead, elements half a tile (two units a thread) ahead.
template <class P, class G, bool SMALL, int GRADS>
__global__ __launch_bounds__(kThreads, 3) void adamw_kernel(const __grid_constant__ StepArgs<GRADS> a) {
    __shared__ union Record {
        uint32_t words[kTileWords];
        Tile tile;
        __device__ Record() {}
    } record[3];
    constexpr int kAcross = kThreads * kSpan, kHalf = 2 * kAcross;
    using Work = Update<P, G, SMALL>;
    const int step = gridDim.x, mine = threadIdx.x * kSpan;
    int index = blockIdx.x;
    const auto word_of = [&](int tile) {
        return threadIdx.x < kTileWords && tile < a.tile_count
                   ? reinterpret_cast<const uint32_t*>(a.tiles + tile)[threadIdx.x]
                   : 0u;
    };
    const auto grad_of = [&](const Tile& t) { return static_cast<const G*>(a.grads[t.tensor - a.first_tensor]) + t.offset; };
    const auto plain = [&](const Tile& t) {  // full and aligned
        return t.count == kTile && t.vector && reinterpret_cast<uintptr_t>(grad_of(t)) % (4 * sizeof(G)) == 0;
    };
    if (threadIdx.x < kTileWords) {
        record[0].words[threadIdx.x] = word_of(index);
        record[1].words[threadIdx.x] = word_of(index + step);
    }
    __syncthreads();
    typename Work::Unit u[2], v[2];
    bool ready = false;  // u holds this tile's first half
    for (int turn = 0; index < a.tile_count; index += step) {
        const uint32_t word = word_of(index + 2 * step);
        const Tile& t = record[turn].tile;
        const int next = turn == 2 ? 0 : turn + 1;
        const Work work{a, t, grad_of(t), 1.0f - a.lr * t.decay};
        if (plain(t)) {
            if (!ready) {
                work.load(u[0], mine, kTile, true, true);
                work.load(u[1], mine + kAcross, kTile, true, true);
            }
            work.load(v[0], mine + kHalf, kTile, true, true);
            work.load(v[1], mine + kHalf + kAcross, kTile, true, true);
            work.finish(u[0], mine, kTile, true);
            work.finish(u[1], mine + kAcross, kTile, true);
            const Tile& n = record[next].tile;
            ready = index + step < a.tile_count && plain(n);
            if (ready) {
                const Work ahead{a, n, grad_of(n), 0.0f};
                ahead.load(u[0], mine, kTile, true, true);
                ahead.load(u[1], mine + kAcross, kTile, true, true);
            }
            work.finish(v[0], mine + kHalf, kTile, true);
            work.finish(v[1], mine + kHalf + kAcross, kTile, true);
        } else {
            const int count = t.count;
            const bool vec_p = t.vector, vec_g = reinterpret_cast<uintptr_t>(work.g) % (4 * sizeof(G)) == 0;
            ready = false;
#pragma unroll 1
            for (int at = mine; at - (int)(threadIdx.x & 31) * kSpan < count; at += kAcross) {  // by warps
                work.load(u[0], at, count, vec_p, vec_g);
                work.finish(u[0], at, count, vec_p);
            }
        }
        if (threadIdx.x < kTileWords) record[next == 2 ? 0 : next + 1].words[threadIdx.x] = word;
        turn = next;
        __syncthreads();
    }
}

}  // namespace

struct mdsoap_adamw {
    std::mutex mutex;
    std::vector<Tensor> tensors;
    std::vector<int64_t> tile_begin;  // [tensors + 1]
    int32_t dtype = 0, state_bits = 32, device = 0;
    uint32_t seed = 0;
    void* table = nullptr;  // the tiles, on `device`
    bool ready = false;     // the table holds them
    ~mdsoap_adamw() {
        if (table) cudaFree(table);
    }
};

namespace {

// Tile records from the tensors and their first tiles ([tensors + 1]).
__global__ void tiles_kernel(const Tensor* tensors, const int64_t* begin, int count, int p_size, int state_size, Tile* out) {
    const int64_t index = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (index >= begin[count]) return;
    int low = 0, high = count;  // the last tensor that begins at or before this tile and has tiles
    while (high - low > 1) {
        const int middle = (low + high) / 2;
        if (begin[middle] <= index) low = middle;
        else high = middle;
    }
    const Tensor t = tensors[low];
    const int64_t at = (index - begin[low]) * kTile;
    out[index] = {t.p + at * p_size,
                  t.m + at * state_size,
                  t.v + at * state_size,
                  t.m_scale ? t.m_scale + at / kBlock : nullptr,
                  t.v_scale ? t.v_scale + at / kBlock : nullptr,
                  t.first + at,
                  at,
                  low,
                  (int32_t)min((int64_t)kTile, t.count - at),
                  t.decay,
                  t.vector};
}

// The table of tiles on the device, made by the first step on its stream.
void upload(mdsoap_adamw& o, cudaStream_t stream) {
    if (o.ready) return;
    if (o.table) cudaFree(o.table), o.table = nullptr;  // of an upload that failed
    const int64_t tiles = o.tile_begin.back();
    const size_t records = tiles * sizeof(Tile), tensors = o.tensors.size() * sizeof(Tensor);
    void* table = nullptr;
    check(engine_malloc(&table, records + tensors + o.tile_begin.size() * sizeof(int64_t)), "optimizer table");
    o.table = table;  // freed with the optimizer
    uint8_t* const device = static_cast<uint8_t*>(table);
    const auto put = [&](size_t at, const void* from, size_t bytes) {
        check(cudaMemcpyAsync(device + at, from, bytes, cudaMemcpyHostToDevice, stream), "optimizer table upload");
    };
    put(records, o.tensors.data(), tensors);  // pageable: copied out before the call returns
    put(records + tensors, o.tile_begin.data(), o.tile_begin.size() * sizeof(int64_t));
    tiles_kernel<<<(unsigned)((tiles + 127) / 128), 128, 0, stream>>>(
        reinterpret_cast<const Tensor*>(device + records), reinterpret_cast<const int64_t*>(device + records + tensors),
        (int)o.tensors.size(), o.dtype == MDSOAP_FLOAT32 ? 4 : 2, o.state_bits / 8, reinterpret_cast<Tile*>(device));
    check(cudaGetLastError(), "optimizer table launch");
    // later steps may come on other streams
    check(cudaStreamSynchronize(stream), "optimizer table");
    o.ready = true;
}

template <class P, class G, int GRADS>
void launch(bool small, const StepSettings& settings, const void* const* grads, size_t count, unsigned grid,
            cudaStream_t stream) {
    StepArgs<GRADS> a;
    static_cast<StepSettings&>(a) = settings;
    std::fill(std::copy_n(grads, count, a.grads), a.grads + GRADS, nullptr);
    if (small) adamw_kernel<P, G, true, GRADS><<<grid, kThreads, 0, stream>>>(a);
    else adamw_kernel<P, G, false, GRADS><<<grid, kThreads, 0, stream>>>(a);
    check(cudaGetLastError(), "optimizer launch");
}

}  // namespace

extern "C" {

int mdsoap_adamw_create(const mdsoap_adamw_params* params, mdsoap_adamw** optimizer) {
    if (!params || !optimizer) return fail(MDSOAP_INVALID_ARGUMENT, "null argument");
    *optimizer = nullptr;
    return entry([&] {
        const mdsoap_adamw_params& q = *params;
        need(q.tensors >= 0 && (q.tensors == 0 || (q.params && q.exp_avg && q.exp_avg_sq && q.counts)),
             "readout: the optimizer needs its tensors");
        need(q.state_bits == 32 || q.state_bits == 8, "readout: optimizer states take 32 or 8 bits");
        need(q.state_bits == 32 || q.tensors == 0 || (q.exp_avg_scale && q.exp_avg_sq_scale),
             "readout: 8-bit optimizer states need their scales");
        by_type(q.dtype, [](auto) {});
        auto o = std::make_unique<mdsoap_adamw>();
        o->dtype = q.dtype;
        o->state_bits = q.state_bits;
        o->seed = q.seed;
        o->device = q.device;
        o->tile_begin.push_back(0);
        int64_t first = 0;
        const uintptr_t p_align = q.dtype == MDSOAP_FLOAT32 ? 16 : 8, state_align = q.state_bits == 32 ? 16 : 4;
        for (int64_t i = 0; i < q.tensors; ++i) {
            Tensor t{};
            t.count = q.counts[i];
            need(t.count >= 0, "readout: negative tensor size");
            t.p = static_cast<uint8_t*>(q.params[i]);
            t.m = static_cast<uint8_t*>(q.exp_avg[i]);
            t.v = static_cast<uint8_t*>(q.exp_avg_sq[i]);
            if (q.state_bits == 8) t.m_scale = q.exp_avg_scale[i], t.v_scale = q.exp_avg_sq_scale[i];
            need(t.count == 0 || (t.p && t.m && t.v && (q.state_bits == 32 || (t.m_scale && t.v_scale))),
                 "readout: null optimizer tensor");
            t.first = first;
            t.decay = q.weight_decay ? q.weight_decay[i] : 0.0f;
            need(t.decay >= 0.0f, "readout: negative weight decay");
            t.vector = (uintptr_t)t.p % p_align == 0 && (uintptr_t)t.m % state_align == 0 &&
                       (uintptr_t)t.v % state_align == 0;
            first += blocks_of(t.count) * kBlock;
            o->tensors.push_back(t);
            o->tile_begin.push_back(o->tile_begin.back() + (t.count + kTile - 1) / kTile);
        }
        need(o->tile_begin.back() <= 0x7fffffff, "readout: too many optimizer elements");
        *optimizer = o.release();
    });
}

void mdsoap_adamw_destroy(mdsoap_adamw* optimizer) { delete optimizer; }

int mdsoap_adamw_step(mdsoap_adamw* optimizer, const void* const* grads, int32_t grad_dtype, int64_t step, double lr,
                      double beta1, double beta2, double eps, double grad_scale, void* stream) {
    if (!optimizer) return fail(MDSOAP_INVALID_ARGUMENT, "null argument");
    return entry([&] {
        mdsoap_adamw& o = *optimizer;
        need(step >= 1, "readout: optimizer steps count from 1");
        need(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "readout: betas must lie in [0, 1)");
        need(lr >= 0.0 && eps >= 0.0 && std::isfinite(lr) && std::isfinite(eps) && std::isfinite(grad_scale),
             "readout: invalid optimizer settings");
        need(grads || o.tensors.empty(), "readout: the optimizer step needs gradients");
        for (size_t i = 0; i < o.tensors.size(); ++i)
            need(grads[i] || o.tensors[i].count == 0, "readout: null gradient");
        by_type(grad_dtype, [](auto) {});
        if (o.tile_begin.back() == 0) return;
        std::lock_guard<std::mutex> lock(o.mutex);
        const OnDevice current(o.device);
        cudaStreamCaptureStatus capture;
        check(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture), "optimizer stream");
        need(capture == cudaStreamCaptureStatusNone,
             "readout: an optimizer step cannot be captured: every replay would be the same step");
        upload(o, static_cast<cudaStream_t>(stream));
        StepSettings a;
        const Tile* tiles = static_cast<const Tile*>(o.table);
        const int sms = sm_count(o.device);
        a.lr = (float)lr;
        a.beta1 = (float)beta1;
        a.beta2 = (float)beta2;
        a.rest1 = (float)(1.0 - beta1);
        a.rest2 = (float)(1.0 - beta2);
        a.eps = (float)eps;
        a.step_size = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
        a.root2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
        a.grad_scale = (float)grad_scale;
        a.key = o.seed * 0x6A09E667u + (uint32_t)step * 0xBB67AE85u;
        for (size_t i = 0; i < o.tensors.size(); i += kGrads) {
            const size_t end = std::min(o.tensors.size(), i + kGrads);
            const int64_t count = o.tile_begin[end] - o.tile_begin[i];
            if (count == 0) continue;
            a.first_tensor = (int32_t)i;
            a.tile_count = (int32_t)count;
            a.tiles = tiles + o.tile_begin[i];
            const unsigned grid = (unsigned)std::min<int64_t>(count, 3 * sms);
            cudaStream_t s = static_cast<cudaStream_t>(stream);
            by_type(o.dtype, [&](auto p) {
                by_type(grad_dtype, [&](auto g) {
                    using P = decltype(p);
                    using G = decltype(g);
                    if (end - i <= kFewGrads) launch<P, G, kFewGrads>(o.state_bits == 8, a, grads + i, end - i, grid, s);
                    else launch<P, G, kGrads>(o.state_bits == 8, a, grads + i, end - i, grid, s);
                });
            });
        }
    });
}

}  // extern "C"
