// Global norm of the gradients of many tensors, and clipping by it (in place, or folded into the optimizer step: param_ops.hip).
// HBM bound for large models (the norm reads every gradient once, clipping reads and writes it once more); for the denoiser's 27 MB
// the launches count, so that a call over up to GC_MAX spans of memory is two launches (beyond that, two for each GC_MAX): the table of spans travels in the
// kernel arguments (no copy to the device, nothing that a captured graph could find changed), and the second launch adds the
// first one's partial sums itself, in every workgroup, instead of waiting for a third.
//   Squares are summed in fp64: the product of two fp32 numbers is exact there, nothing finite overflows, and the cost hides
// behind the loads.  Partial sums are added in a fixed order.
#include <type_traits>
#include "common.h"
#include "ddpm_hip.h"

typedef _Float16 f16;

namespace {
constexpr int GC_MAX = 320;                 // spans per launch: 12 bytes each of the 4 KB that kernel arguments may take
constexpr int GC_THREADS = 1024;
constexpr int GC_CHUNK = 2 * GC_THREADS;    // 16-byte vectors a workgroup takes at once
constexpr int GC_GRID = 512;                // two workgroups of 16 waves per CU: every wave the card can hold
constexpr int GC_INLINE = 8 * GC_GRID;      // most partial sums that each workgroup of the second launch adds up by itself

struct GcSpans {
    uint64_t at[GC_MAX];                    // address; the element type in the two highest bits
    uint32_t n[GC_MAX];
    int count;
};
}  // namespace

// one element as it counts for the norm: |g| as raw bits for the maximum (NaN is larger than infinity there), g^2 for the sum
__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

struct GcAcc {
    double sum;
    uint32_t top;
};

template <bool INF> __device__ __forceinline__ void gc_add(GcAcc& a, float f) {
    if (INF) {
        const uint32_t b = abs_bits(f);
        a.top = a.top > b ? a.top : b;
    } else {
        const double d = (double)f;
        a.sum = fma(d, d, a.sum);
    }
}
// (LDS: one entry per wave; every thread returns the workgroup's value, waves combined in ascending order)
template <bool INF> __device__ __forceinline__ GcAcc gc_block(GcAcc a, GcAcc* s) {
    for (int o = 32; o > 0; o >>= 1) {
        if (INF) {
            const uint32_t b = __shfl_xor(a.top, o, 64);
            a.top = a.top > b ? a.top : b;
        } else
            a.sum += __shfl_xor(a.sum, o, 64);
    }
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a;
    __syncthreads();
    GcAcc r = s[0];
#pragma unroll
    for (int k = 1; k < GC_THREADS / 64; ++k) {
        r.sum += s[k].sum;
        r.top = r.top > s[k].top ? r.top : s[k].top;
    }
    __syncthreads();
    return r;
}
template <bool INF> __device__ __forceinline__ float gc_norm_of(const GcAcc& a) { return INF ? __uint_as_float(a.top) : (float)sqrt(a.sum); }

// The part of the span's vectors [v0, v0 + GC_CHUNK) that thread tid sees: f(vector, first element, number of vectors in range).
// A span starts `lead` elements into its first 16-byte vector; vectors that the span covers whole are moved at once, the (at most
// two) others element by element.
template <typename T, typename F1, typename FV>
__device__ __forceinline__ void gc_chunk(T* base, uint32_t n, uint32_t chunk, FV&& whole, F1&& one) {
    constexpr int V = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V)));
    const uint32_t lead = (uint32_t)((uintptr_t)base % 16 / sizeof(T));
    const uint64_t vecs = ((uint64_t)n + lead + V - 1) / V;
    vec* const vbase = (vec*)(base - lead);
#pragma unroll
    for (int k = 0; k < GC_CHUNK / GC_THREADS; ++k) {
        const uint64_t v = (uint64_t)chunk * GC_CHUNK + k * GC_THREADS + threadIdx.x;
        if (v >= vecs) continue;
        const int64_t e = (int64_t)v * V - lead;
        if (e >= 0 && e + V <= (int64_t)n) whole(vbase + v);
        else
            for (int j = 0; j < V; ++j)
                if (e + j >= 0 && e + j < (int64_t)n) one(base + (e + j));
    }
}

// span and chunk of the workgroup's c-th piece of work; first[i]: chunks in front of span i (LDS)
__device__ __forceinline__ int gc_span_of(const uint32_t* first, int count, uint32_t c) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ uint32_t gc_chunks_of(uint64_t at, uint32_t n) {
    const int size = (at >> 62) == DDPM_F32 ? 4 : 2, V = 16 / size;
    return (uint32_t)(((uint64_t)n + (at % 16) / size + V - 1) / V + GC_CHUNK - 1) / GC_CHUNK;
}

// first[0 .. count]: running number of chunks (LDS, GC_MAX + 1 entries); one wave scans five entries a lane
__device__ __forceinline__ void gc_prefix(const GcSpans& sp, uint32_t* first) {
    if (threadIdx.x < 64) {
        constexpr int PER = GC_MAX / 64;
        uint32_t mine[PER], sum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x * PER + j;
            mine[j] = sum;
            sum += i < sp.count ? gc_chunks_of(sp.at[i], sp.n[i]) : 0;
        }
        uint32_t run = sum;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t below = __shfl_up(run, o, 64);
            if ((int)threadIdx.x >= o) run += below;
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) first[threadIdx.x * PER + j] = run - sum + mine[j];
        if (threadIdx.x == 63) first[GC_MAX] = run;
    }
    __syncthreads();
}

template <bool INF> __global__ __launch_bounds__(GC_THREADS) void grad_norm_kernel(const GcSpans sp, GcAcc* __restrict__ part) {
    __shared__ uint32_t first[GC_MAX + 1];
    __shared__ GcAcc s_acc[GC_THREADS / 64];
    gc_prefix(sp, first);
    GcAcc acc = {0.0, 0u};
    for (uint32_t c = blockIdx.x; c < first[GC_MAX]; c += gridDim.x) {
        const int i = gc_span_of(first, sp.count, c);
        const uint64_t at = sp.at[i] & ~(3ull << 62);
        const uint32_t n = sp.n[i], chunk = c - first[i];
        auto run = [&](auto* base) {
            typedef typename std::remove_reference<decltype(*base)>::type T;
            constexpr int V = 16 / sizeof(T);
            typedef T vec __attribute__((ext_vector_type(V)));
            gc_chunk(base, n, chunk, [&](vec* p) {
                const vec x = *p;
#pragma unroll
                for (int j = 0; j < V; ++j) gc_add<INF>(acc, (float)x[j]);
            }, [&](T* p) { gc_add<INF>(acc, (float)*p); });
        };
        const int type = (int)(sp.at[i] >> 62);
        if (type == DDPM_F32) run((float*)at);
        else if (type == DDPM_BF16) run((bf16*)at);
        else run((f16*)at);
    }
    acc = gc_block<INF>(acc, s_acc);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

template <bool INF> __device__ __forceinline__ float gc_total(const GcAcc* part, int parts, GcAcc* s_acc) {
    GcAcc acc = {0.0, 0u};
    for (int k = threadIdx.x; k < parts; k += GC_THREADS) {
        const GcAcc p = part[k];
        acc.sum += p.sum;
        acc.top = acc.top > p.top ? acc.top : p.top;
    }
    return gc_norm_of<INF>(gc_block<INF>(acc, s_acc));
}

template <bool INF> __global__ __launch_bounds__(GC_THREADS) void grad_norm_total_kernel(const GcAcc* __restrict__ part, int parts, float* __restrict__ norm) {
    __shared__ GcAcc s_acc[GC_THREADS / 64];
    const float r = gc_total<INF>(part, parts, s_acc);
    if (threadIdx.x == 0) *norm = r;
}

// parts > 0: the norm is still in partial sums; workgroup 0 of the launch that says so also writes it down
template <bool INF> __global__ __launch_bounds__(GC_THREADS) void grad_scale_kernel(const GcSpans sp, const GcAcc* __restrict__ part, int parts, int write,
                                                                                     float* __restrict__ norm, float max_norm) {
    __shared__ uint32_t first[GC_MAX + 1];
    __shared__ GcAcc s_acc[GC_THREADS / 64];
    gc_prefix(sp, first);
    float total;
    if (parts > 0) {
        total = gc_total<INF>(part, parts, s_acc);
        if (write && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
    } else
        total = *norm;
    const float ratio = max_norm / (total + 1e-6f), coef = ratio > 1.f ? 1.f : ratio;      // (a NaN stays one)
    for (uint32_t c = blockIdx.x; c < first[GC_MAX]; c += gridDim.x) {
        const int i = gc_span_of(first, sp.count, c);
        const uint64_t at = sp.at[i] & ~(3ull << 62);
        const uint32_t n = sp.n[i], chunk = c - first[i];
        auto run = [&](auto* base) {
            typedef typename std::remove_reference<decltype(*base)>::type T;
            constexpr int V = 16 / sizeof(T);
            typedef T vec __attribute__((ext_vector_type(V)));
            // A bf16 tensor is multiplied by the factor rounded to bf16, as torch.nn.utils.clip_grad_norm_ multiplies it: the bits of
            // that, off by at most 2^-8 in a factor common to the whole tensor (and the clipped norm may pass the limit by that).  (An fp16 one is not: fp16 loses factors below 2^-14.)
            const float by = std::is_same<T, bf16>::value ? (float)(bf16)coef : coef;
            gc_chunk(base, n, chunk, [&](vec* p) {
                vec x = *p;
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] = (T)((float)x[j] * by);
                *p = x;
            }, [&](T* p) { *p = (T)((float)*p * by); });
        };
        const int type = (int)(sp.at[i] >> 62);
        if (type == DDPM_F32) run((float*)at);
        else if (type == DDPM_BF16) run((bf16*)at);
        else run((f16*)at);
    }
}

namespace {
constexpr int64_t GC_SPLIT = 1ll << 31;      // a larger tensor is several spans

// calls f(spans, chunks) for every launch's worth of spans; empty tensors take no span
template <typename F>
void gc_for_launches(const uint64_t* ptr, const int64_t* numel, const uint8_t* dtype, int count, F&& f) {
    GcSpans sp;
    sp.count = 0;
    uint64_t chunks = 0;
    auto flush = [&]() {
        if (sp.count) f(sp, chunks);
        sp.count = 0;
        chunks = 0;
    };
    for (int i = 0; i < count; ++i) {
        const int size = dtype[i] == DDPM_F32 ? 4 : 2;
        for (int64_t at = 0; at < numel[i]; at += GC_SPLIT) {
            const int64_t n = numel[i] - at < GC_SPLIT ? numel[i] - at : GC_SPLIT;
            const uint64_t p = ptr[i] + (uint64_t)at * size;
            const int V = 16 / size;
            const uint64_t c = ((uint64_t)n + (p % 16) / size + V - 1) / V / GC_CHUNK + 1;
            if (sp.count == GC_MAX || chunks + c > 0x7fffffffull) flush();
            sp.at[sp.count] = p | (uint64_t)dtype[i] << 62;
            sp.n[sp.count++] = (uint32_t)n;
            chunks += c;
        }
    }
    flush();
}
}  // namespace

extern "C" int64_t ddpm_grad_norm_work_bytes(int count, const int64_t* numel) {
    if (count < 0 || (count > 0 && !numel)) return -1;
    int64_t spans = 0;
    for (int i = 0; i < count; ++i) spans += numel[i] > 0 ? (numel[i] + GC_SPLIT - 1) / GC_SPLIT : 0;
    return ((spans + GC_MAX - 1) / GC_MAX + 1) * GC_GRID * (int64_t)sizeof(GcAcc);
}

extern "C" int ddpm_grad_norm(const uint64_t* ptr, const int64_t* numel, const uint8_t* dtype, int count, int norm_type, int clip, float max_norm,
                              float* norm, void* work, ddpm_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    DDPM_REQUIRE(count >= 0 && (count == 0 || (ptr && numel && dtype)), "grad_norm: null table");
    DDPM_REQUIRE(norm && work, "grad_norm: null pointer");
    DDPM_REQUIRE(norm_type == DDPM_NORM_L2 || norm_type == DDPM_NORM_INF, "grad_norm: unknown norm %d", norm_type);
    DDPM_REQUIRE(!clip || max_norm >= 0.f, "grad_norm: max_norm must not be negative");
    for (int i = 0; i < count; ++i) {
        DDPM_REQUIRE(dtype[i] <= DDPM_F32, "grad_norm: tensor %d has an unknown element type %d", i, dtype[i]);
        DDPM_REQUIRE(numel[i] >= 0 && (numel[i] == 0 || ptr[i]) && ptr[i] >> 62 == 0, "grad_norm: tensor %d is not there", i);
        DDPM_REQUIRE(ptr[i] % (dtype[i] == DDPM_F32 ? 4 : 2) == 0, "grad_norm: tensor %d is not aligned to its element type", i);
    }
    const bool inf = norm_type == DDPM_NORM_INF;
    GcAcc* const part = (GcAcc*)work;
    int parts = 0, launches = 0;
    gc_for_launches(ptr, numel, dtype, count, [&](const GcSpans& sp, uint64_t chunks) {
        const int grid = (int)(chunks < GC_GRID ? chunks : GC_GRID);
        if (inf) hipLaunchKernelGGL(grad_norm_kernel<true>, dim3((unsigned)grid), dim3(GC_THREADS), 0, stream, sp, part + parts);
        else hipLaunchKernelGGL(grad_norm_kernel<false>, dim3((unsigned)grid), dim3(GC_THREADS), 0, stream, sp, part + parts);
        parts += grid;
        ++launches;
    });
    // One sum of the partial sums for everybody where there are so many that adding them in every workgroup would cost more than a launch
    const bool own = !clip || parts == 0 || parts > GC_INLINE;
    if (own) {
        if (inf) hipLaunchKernelGGL(grad_norm_total_kernel<true>, dim3(1), dim3(GC_THREADS), 0, stream, part, parts, norm);
        else hipLaunchKernelGGL(grad_norm_total_kernel<false>, dim3(1), dim3(GC_THREADS), 0, stream, part, parts, norm);
    }
    if (clip) {
        int done = 0;
        gc_for_launches(ptr, numel, dtype, count, [&](const GcSpans& sp, uint64_t chunks) {
            const int grid = (int)(chunks < GC_GRID ? chunks : GC_GRID);
            if (inf) hipLaunchKernelGGL(grad_scale_kernel<true>, dim3((unsigned)grid), dim3(GC_THREADS), 0, stream, sp, part, own ? 0 : parts, done == 0, norm, max_norm);
            else hipLaunchKernelGGL(grad_scale_kernel<false>, dim3((unsigned)grid), dim3(GC_THREADS), 0, stream, sp, part, own ? 0 : parts, done == 0, norm, max_norm);
            ++done;
        });
    }
    return ddpm_check_launch("grad_norm");
}
