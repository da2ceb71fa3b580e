// Layer norm over the last axis of token rows, forward and backward, next to the per-sample GroupNorm(1, C) of attention.hip:
//   y = (x - mu) * rstd * w + b                        mu, rstd of each row
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat))  g = dy * w, xhat = (x - mu) * rstd
//   dw = sum over rows of dy * xhat, db = sum over rows of dy
// Both passes move every element once (x -> y; x, dy -> dx) and are bound by HBM: a row lives in registers between its loads and
// its store, and w, b and the column sums of dw, db live in registers across the rows that a workgroup works through, so that
// neither the parameters nor a second sweep over x and dy cost bandwidth (16384 x 1024 bf16: 15 us forward, 28 backward with the sums;
// 14 and 21 at the rate of a large copy).  The next row's loads are issued before the current
// row's reduction.  Rows of up to 1024 elements belong to a group of 4 ... 64 lanes of one wave (reduction by lane exchanges
// only), longer ones to a workgroup of 256 or 512 threads (one barrier per row).
//   Statistics: mean first, then squared deviations from it, both from the registers, in fp32: no difference of large sums.  Across
// waves: sum n_w (mean_w - mean)^2 + M2_w, which has no cancellation either.
//   Column sums: each workgroup writes one row [2][C] of partial sums, a second launch adds the rows in a fixed order, so that
// the gradients of the parameters are the same numbers in every run.
#include "common.h"
#include "ddpm_hip.h"

typedef _Float16 f16;

template <typename T, int N> struct VecOf { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct VecOf<T, 1> { typedef T type; };
template <typename T, int V> __device__ __forceinline__ float vec_get(const typename VecOf<T, V>::type& v, int j) {
    if constexpr (V == 1) return (float)v;
    else return (float)v[j];
}
template <typename T, int V> __device__ __forceinline__ void vec_set(typename VecOf<T, V>::type& v, int j, float f) {
    if constexpr (V == 1) v = (T)f;
    else v[j] = (T)f;
}

// N consecutive floats at any multiple of 4 bytes
template <int N> __device__ __forceinline__ void ln_get(float* f, const float* p) {
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const vec v = *(const vec*)(p + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[j + i] = v[i];
        }
    } else
        f[0] = *p;
}
template <int N> __device__ __forceinline__ void ln_put(float* p, const float* f) {
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 4) *(vec*)(p + j) = vec{f[j], f[j + 1], f[j + 2], f[j + 3]};
    } else
        *p = f[0];
}

struct LnArgs {
    const void *x, *dy;
    void *y, *dx;
    const float *w, *b;
    float *stats, *part;       // [rows][2] (mean, rstd); [gridDim.x][2][C]
    long long rows, ldx, ldy, lddy, lddx;
    int C, tpr;                // threads per row where a row is a part of a wave
    float eps, inv_c;
};

__device__ __forceinline__ float group_sum(float v, int tpr) {
    for (int o = 1; o < tpr; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Thread t of the tpr threads of a row holds elements (v * tpr + t) * V ... + V-1, v < NV.
template <typename T, int V, int NV, int BLOCK>
__global__ __launch_bounds__(BLOCK ? BLOCK : 256) void ln_fwd_kernel(const LnArgs a) {
    typedef typename VecOf<T, V>::type vec;
    constexpr int WAVES = BLOCK ? BLOCK / 64 : 1;
    __shared__ float2 s_red[2][WAVES];
    const int tid = threadIdx.x, tpr = BLOCK ? BLOCK : a.tpr, t = BLOCK ? tid : tid & (tpr - 1);
    const long long step = BLOCK ? gridDim.x : (long long)gridDim.x * (256 / tpr);
    const T* const x = (const T*)a.x;
    T* const y = (T*)a.y;
    float w[NV * V], b[NV * V];
    int count = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * tpr + t) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) { w[v * V + j] = 1.f; b[v * V + j] = 0.f; }
        if (c < a.C) {
            if (a.w) ln_get<V>(w + v * V, a.w + c);
            if (a.b) ln_get<V>(b + v * V, a.b + c);
            count += V;
        }
    }
    // the wave's share of a row: its size (LDS: of every wave) and reciprocal
    __shared__ float s_n[WAVES];
    const float n_w = BLOCK ? group_sum((float)count, 64) : 0.f, inv_n = n_w > 0.f ? 1.f / n_w : 0.f;
    if (BLOCK && (tid & 63) == 0) s_n[tid >> 6] = n_w;             // (read behind the barrier of the first row)
    vec next[NV];
    auto fetch = [&](long long row) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * tpr + t) * V;
            if (c < a.C) next[v] = *(const vec*)(x + row * a.ldx + c);
        }
    };
    const long long row0 = BLOCK ? blockIdx.x : (long long)blockIdx.x * (256 / tpr) + tid / tpr;
    // (a group of lanes past the last row repeats it, so that the lanes of a wave stay together, and stores nothing)
    fetch(row0 < a.rows ? row0 : a.rows - 1);
    int parity = 0;
    for (long long row = row0, first = BLOCK ? row0 : (long long)blockIdx.x * (256 / tpr); first < a.rows; row += step, first += step, parity ^= 1) {
        float f[NV * V];
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < V; ++j) f[v * V + j] = (v * tpr + t) * V + j < a.C ? vec_get<T, V>(next[v], j) : 0.f;
        if (first + step < a.rows) fetch(row + step < a.rows ? row + step : a.rows - 1);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV * V; ++i) s += f[i];
        float mean = group_sum(s, BLOCK ? 64 : tpr) * (BLOCK ? inv_n : a.inv_c), q = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = (v * tpr + t) * V + j < a.C ? f[v * V + j] - mean : 0.f;
                q += d * d;
            }
        q = group_sum(q, BLOCK ? 64 : tpr);
        if constexpr (BLOCK != 0) {
            // (mean of the wave's share, squared deviations from it)
            if ((tid & 63) == 0) s_red[parity][tid >> 6] = make_float2(mean, q);
            __syncthreads();
            float total = 0.f, dev = 0.f;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) total += s_red[parity][k].x * s_n[k];
            total *= a.inv_c;
            q = 0.f;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) {
                const float2 r = s_red[parity][k];
                dev += s_n[k] * (r.x - total) * (r.x - total);
                q += r.y;
            }
            q += dev;
            mean = total;
        }
        const float rstd = rsqrtf(q * a.inv_c + a.eps);
        if (row < a.rows) {
            if (a.stats && t == 0) *(float2*)(a.stats + 2 * row) = make_float2(mean, rstd);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * tpr + t) * V;
                vec o;
#pragma unroll
                for (int j = 0; j < V; ++j) vec_set<T, V>(o, j, (f[v * V + j] - mean) * rstd * w[v * V + j] + b[v * V + j]);
                if (c < a.C) *(vec*)(y + row * a.ldy + c) = o;
            }
        }
    }
}

template <typename T, int V, int NV, int BLOCK>
__global__ __launch_bounds__(BLOCK ? BLOCK : 256) void ln_bwd_kernel(const LnArgs a) {
    typedef typename VecOf<T, V>::type vec;
    constexpr int WAVES = BLOCK ? BLOCK / 64 : 1, E = NV * V;
    extern __shared__ float s_col[];                 // wave rows: [4][2][C], the waves' column sums
    __shared__ float2 s_red[2][WAVES];
    const int tid = threadIdx.x, tpr = BLOCK ? BLOCK : a.tpr, t = BLOCK ? tid : tid & (tpr - 1);
    const long long step = BLOCK ? gridDim.x : (long long)gridDim.x * (256 / tpr);
    const T *const x = (const T*)a.x, *const dy = (const T*)a.dy;
    T* const dx = (T*)a.dx;
    float w[E], dw[E], db[E];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * tpr + t) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) { w[v * V + j] = 1.f; dw[v * V + j] = db[v * V + j] = 0.f; }
        if (a.w && c < a.C) ln_get<V>(w + v * V, a.w + c);
    }
    vec nx[NV], nd[NV];
    float2 nst = make_float2(0.f, 0.f);
    auto fetch = [&](long long row) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * tpr + t) * V;
            if (c < a.C) {
                nx[v] = *(const vec*)(x + row * a.ldx + c);
                nd[v] = *(const vec*)(dy + row * a.lddy + c);
            }
        }
        nst = *(const float2*)(a.stats + 2 * row);
    };
    const long long block0 = BLOCK ? blockIdx.x : (long long)blockIdx.x * (256 / tpr);
    const long long row0 = BLOCK ? block0 : block0 + tid / tpr;
    fetch(row0 < a.rows ? row0 : a.rows - 1);
    int parity = 0;
    for (long long row = row0, first = block0; first < a.rows; row += step, first += step, parity ^= 1) {
        const bool live = row < a.rows;
        const float mean = nst.x, rstd = nst.y;
        float h[E], g[E], c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const bool in = (i / V * tpr + t) * V + i % V < a.C && live;
            h[i] = in ? (vec_get<T, V>(nx[i / V], i % V) - mean) * rstd : 0.f;
            const float d = in ? vec_get<T, V>(nd[i / V], i % V) : 0.f;
            dw[i] += d * h[i];
            db[i] += d;
            g[i] = d * w[i];
            c1 += g[i];
            c2 += g[i] * h[i];
        }
        if (first + step < a.rows) fetch(row + step < a.rows ? row + step : a.rows - 1);
        c1 = group_sum(c1, BLOCK ? 64 : tpr);
        c2 = group_sum(c2, BLOCK ? 64 : tpr);
        if constexpr (BLOCK != 0) {
            if ((tid & 63) == 0) s_red[parity][tid >> 6] = make_float2(c1, c2);
            __syncthreads();
            c1 = c2 = 0.f;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) { c1 += s_red[parity][k].x; c2 += s_red[parity][k].y; }
        }
        c1 *= a.inv_c;
        c2 *= a.inv_c;
        if (live && a.dx) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * tpr + t) * V;
                vec o;
#pragma unroll
                for (int j = 0; j < V; ++j) vec_set<T, V>(o, j, rstd * (g[v * V + j] - c1 - h[v * V + j] * c2));
                if (c < a.C) *(vec*)(dx + row * a.lddx + c) = o;
            }
        }
    }
    if (!a.part) return;
    float* const part = a.part + (long long)blockIdx.x * 2 * a.C;
    if constexpr (BLOCK != 0) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * tpr + t) * V;
            if (c < a.C) {
                ln_put<V>(part + c, dw + v * V);
                ln_put<V>(part + a.C + c, db + v * V);
            }
        }
    } else {
        // lane groups of the wave, then the four waves through LDS, each in a fixed order
        float* const mine = s_col + (tid >> 6) * 2 * a.C;
#pragma unroll
        for (int i = 0; i < E; ++i)
            for (int o = tpr; o < 64; o <<= 1) { dw[i] += __shfl_xor(dw[i], o, 64); db[i] += __shfl_xor(db[i], o, 64); }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * tpr + t) * V;
            if ((tid & 63) < tpr && c < a.C) {
                ln_put<V>(mine + c, dw + v * V);
                ln_put<V>(mine + a.C + c, db + v * V);
            }
        }
        __syncthreads();
        for (int i = tid; i < 2 * a.C; i += 256) part[i] = (s_col[i] + s_col[2 * a.C + i]) + (s_col[4 * a.C + i] + s_col[6 * a.C + i]);
    }
}

// out[c] = sum over the rows of part: a workgroup takes 64 of the 2C columns, its 16 waves every 16th row
__global__ __launch_bounds__(1024) void ln_param_grad_kernel(const float* __restrict__ part, int rows, int C, float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float s[16][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = blockIdx.x * 64 + lane;
    float acc = 0.f;
    if (c < 2 * C) {
#pragma unroll 8
        for (int r = wave; r < rows; r += 16) acc += part[(long long)r * 2 * C + c];
    }
    s[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && c < 2 * C) {
#pragma unroll
        for (int k = 1; k < 16; ++k) acc += s[k][lane];
        float* const out = c < C ? dw : db;
        if (out) out[c < C ? c : c - C] = acc;
    }
}

// ---- launch ----------------------------------------------------------------------------------------------------------------
namespace {
struct LnPlan { int vec, nv, block, tpr, grid; };

constexpr int LN_MAX_C = 8192;

// Elements per thread: at most 16, so that parameters, sums and two rows in flight fit the registers without spilling.
bool ln_plan(long long rows, int C, bool aligned, int size, bool fwd, LnPlan& p) {
    const int V = aligned ? 16 / size : 1;
    p.vec = V;
    const int vecs = (C + V - 1) / V, most = 16 / V;                   // vectors in a row, vectors per thread
    p.block = vecs <= 64 * most ? 0 : vecs <= 256 * most ? 256 : 512;
    if (p.block == 0) {
        p.tpr = 4;
        while (p.tpr < 64 && p.tpr < vecs) p.tpr *= 2;
    } else
        p.tpr = p.block;
    const int need = (vecs + p.tpr - 1) / p.tpr;
    p.nv = 1;
    while (p.nv < need) p.nv *= 2;
    const long long groups = p.block ? rows : (rows + 256 / p.tpr - 1) / (256 / p.tpr);
    // Workgroups per CU: enough loads in flight for HBM, but each begins with w, b (and ends with the column sums), which the rows it works
    // through have to pay for.  us at 65536 x 4096 bf16: forward 218 / 200 / 182 with 6 / 3 / 2 a CU, but 59 / 49 / 60 at 20000 x 3000; a wave to
    // a row, 65536 x 512: 37 / 28 / 28 with 3 / 6 / 8.  Backward, 65536 x 4096: 337 / 293 with 4 / 2; 8192 x 8192: 86 / 80 with 2 / 1; a wave to a
    // row of 16384 x 1024: 34 / 28 with 4 / 2, of 65536 x 512: 45 / 58.
    const int per_cu = fwd ? (p.block == 0 ? 6 : p.block == 256 ? 3 : 2) : p.block == 512 ? 1 : p.block == 256 || p.nv * V == 16 ? 2 : 4;
    const long long cap = 256 * per_cu;
    p.grid = (int)(groups < cap ? groups : cap);
    return p.nv <= most;
}

// (a workgroup of 256 is taken for rows that fill more than a quarter of it, one of 512 for rows that fill more than half)
template <typename T, int V, int NV, bool FWD>
void ln_launch_nv(const LnPlan& p, const LnArgs& a, hipStream_t st) {
    constexpr int MOST = 16 / V;
    const dim3 grid((unsigned)p.grid);
    if (p.block == 0) {
        if constexpr (FWD) hipLaunchKernelGGL((ln_fwd_kernel<T, V, NV, 0>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((ln_bwd_kernel<T, V, NV, 0>), grid, dim3(256), a.part ? 32 * a.C : 0, st, a);
    } else if (p.block == 256) {
        if constexpr (NV * 2 >= MOST) {
            if constexpr (FWD) hipLaunchKernelGGL((ln_fwd_kernel<T, V, NV, 256>), grid, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((ln_bwd_kernel<T, V, NV, 256>), grid, dim3(256), 0, st, a);
        }
    } else {
        if constexpr (NV == MOST) {
            if constexpr (FWD) hipLaunchKernelGGL((ln_fwd_kernel<T, V, NV, 512>), grid, dim3(512), 0, st, a);
            else hipLaunchKernelGGL((ln_bwd_kernel<T, V, NV, 512>), grid, dim3(512), 0, st, a);
        }
    }
}

template <typename T, int V, bool FWD>
void ln_launch_v(const LnPlan& p, const LnArgs& a, hipStream_t st) {
    switch (p.nv) {
        case 1: ln_launch_nv<T, V, 1, FWD>(p, a, st); break;
        case 2: ln_launch_nv<T, V, 2, FWD>(p, a, st); break;
        case 4: if constexpr (V <= 4) ln_launch_nv<T, V, 4, FWD>(p, a, st); break;
        case 8: if constexpr (V <= 2) ln_launch_nv<T, V, 8, FWD>(p, a, st); break;
        default: if constexpr (V == 1) ln_launch_nv<T, V, 16, FWD>(p, a, st); break;
    }
}

template <typename T, bool FWD>
void ln_launch(const LnPlan& p, const LnArgs& a, hipStream_t st) {
    if (p.vec == 1) ln_launch_v<T, 1, FWD>(p, a, st);
    else ln_launch_v<T, 16 / sizeof(T), FWD>(p, a, st);
}

int ln_setup(const ddpm_layer_norm_desc* d, bool fwd, LnPlan& p) {
    DDPM_REQUIRE(d, "layer_norm: null descriptor");
    DDPM_REQUIRE(d->dtype >= DDPM_BF16 && d->dtype <= DDPM_F32, "layer_norm: unknown element type %d", d->dtype);
    DDPM_REQUIRE(d->rows >= 0 && d->C >= 1 && d->C <= LN_MAX_C, "layer_norm: %lld rows of %d elements (1 to %d)", (long long)d->rows, d->C, LN_MAX_C);
    DDPM_REQUIRE(d->eps >= 0.f, "layer_norm: eps must not be negative");
    if (d->rows == 0) return DDPM_OK;
    DDPM_REQUIRE(d->x && (fwd ? d->y != nullptr : d->dy && d->stats), "layer_norm: null pointer");
    DDPM_REQUIRE(d->rows == 1 || (d->ldx >= d->C && (fwd ? d->ldy >= d->C : d->lddy >= d->C && (!d->dx || d->lddx >= d->C))),
                 "layer_norm: a row stride is shorter than a row");
    const int size = d->dtype == DDPM_F32 ? 4 : 2, V = 16 / size;
    auto fits = [&](const void* q, int64_t ld) { return !q || ((uintptr_t)q % 16 == 0 && (d->rows == 1 || ld % V == 0)); };
    const bool aligned = d->C % V == 0 && fits(d->x, d->ldx) && (fwd ? fits(d->y, d->ldy) : fits(d->dy, d->lddy) && fits(d->dx, d->lddx));
    DDPM_REQUIRE(ln_plan(d->rows, d->C, aligned, size, fwd, p), "layer_norm: no plan for %d elements", d->C);
    return DDPM_OK;
}

template <bool FWD>
int ln_run(const ddpm_layer_norm_desc* d, hipStream_t st) {
    LnPlan p = {};
    if (const int rc = ln_setup(d, FWD, p)) return rc;
    const bool params = !FWD && (d->dw || d->db);
    DDPM_REQUIRE(!params || d->rows == 0 || d->part, "layer_norm: the parameters' gradients need the workspace `part`");
    if (d->rows > 0) {
        LnArgs a = {d->x, d->dy, d->y, d->dx, d->w, d->b, d->stats, params ? d->part : nullptr, d->rows, d->ldx, d->ldy, d->lddy, d->lddx, d->C,
                    p.tpr, d->eps, 1.0f / (float)d->C};
        if (d->dtype == DDPM_BF16) ln_launch<bf16, FWD>(p, a, st);
        else if (d->dtype == DDPM_F16) ln_launch<f16, FWD>(p, a, st);
        else ln_launch<float, FWD>(p, a, st);
    }
    if (params)
        hipLaunchKernelGGL(ln_param_grad_kernel, dim3((unsigned)((2 * d->C + 63) / 64)), dim3(1024), 0, st, d->part, p.grid, d->C, d->dw, d->db);
    else if (d->rows == 0)
        return DDPM_OK;
    return ddpm_check_launch(FWD ? "layer_norm_forward" : "layer_norm_backward");
}
}  // namespace

extern "C" int ddpm_layer_norm_part_rows(const ddpm_layer_norm_desc* d) {
    LnPlan p = {};
    return ln_setup(d, false, p) == DDPM_OK ? p.grid : -1;
}
extern "C" int ddpm_layer_norm_forward(const ddpm_layer_norm_desc* d, ddpm_stream_t stream) { return ln_run<true>(d, (hipStream_t)stream); }
extern "C" int ddpm_layer_norm_backward(const ddpm_layer_norm_desc* d, ddpm_stream_t stream) { return ln_run<false>(d, (hipStream_t)stream); }
