// Attention over packed sequences of different lengths, causal or not, with grouped heads and an optional learned relative
// position bias; forward and backward.  (attention.hip next to it serves ConditionalModule: batches of one length, head widths to
// 64, every key in LDS, dropout.)
//   s_ij = scale * q_i . k_j + table[bucket(j - i), head]      p = softmax over the keys j that query i sees      o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i      ds_ij = p_ij (do_i . v_j - D_i), D_i = do_i . o_i      dq_i = scale sum_j ds_ij k_j
//   dk_j = scale sum_i ds_ij q_i (over every head that shares k_j)      dtable[b, head] = sum of ds_ij over the pairs with bucket b
// The product of each head's width with every visible pair is what it cannot do without: the matrix cores bound it for wide
// heads, the exponentials for narrow ones.
//
// Tiles.  A workgroup is four waves; a wave owns 32 rows of the output (queries; keys for dk, dv), and the four share tiles of 64
// rows of the other side in LDS, two buffers of them, the next tile's global loads in flight in registers during the current
// one's products: one barrier per tile.  Every product is arranged so that the OWNED row is a COLUMN of the matrix result
// (v_mfma_f32_32x32x16: lane l holds column l % 32, register i row (i/4)*8 + (l/32)*4 + i%4), i.e. s^T = k q^T, o^T = v^T p^T.
// The running maximum and sum of a row are then one number per lane, and the probabilities go from result registers to the next
// product's operand without leaving the lane (a contraction may be permuted as long as both operands agree).  The other
// operand of that product is read transposed from the same LDS tile (ds_read_b64_tr_b16).  Rows of a tile are stored with their 16-byte
// pieces exchanged by a row-dependent xor, so that the lanes of either kind of read fall on different banks.
//
// Sequences.  The launch has one slot for every 128 rows plus one per sequence: floor(begin / 128) + index never collides and needs no
// host knowledge of the lengths.  A workgroup finds its sequence from the boundaries by one load and a ballot.  Rows outside of all
// sequences are two more sequences without keys: their results are zeros where the caller wants that, and they are not touched otherwise.
// Boundaries are clamped to the tensors, so that no contents of that array reach outside of them.
#include <type_traits>
#include "common.h"
#include "ddpm_hip.h"

typedef _Float16 f16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

#define PA_ROWS 128          /* rows of a workgroup */
#define PA_TILE 64           /* rows of a tile of the other side */

struct PaView {              // element (row, head, d) at p[row * row_stride + head * head_stride + d]
    void* p;
    long long row, head;
};

struct PaArgs {
    PaView q, k, v, o, dout, dq, dk, dv;
    float *o32, *lse, *dsum;                 // [Tq][H][dh]; [H][Tq] each
    const int *ends_q, *ends_k;              // [B + 1]
    const float* table;                      // [buckets][H]
    const int* bucket_of;                    // [2 * far + 1]
    float* dtable_part;                      // [slots][H][buckets]
    int buckets, far;
    int Tq, Tk, B, H, Hk, dh, causal, zero_rest, slots;
    float scale, scale2;                     // and times log2(e)
};

__device__ __forceinline__ f32x16 pa_mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 pa_mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

template <typename T> struct PaTypes;
template <> struct PaTypes<bf16> { typedef bf16x8 v8; typedef bf16x4 v4; };
template <> struct PaTypes<f16> { typedef f16x8 v8; typedef f16x4 v4; };

__device__ __forceinline__ f32x16 pa_zero() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}
// the other half-wave's value combined with this one's: both halves hold the result
__device__ __forceinline__ float pa_half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pa_half_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- sequences ---------------------------------------------------------------------------------------------------------------
struct PaSeq {
    int begin, n;            // rows of the side that the launch's slots run over
    int begin2, n2;          // rows of the other side
    int row0;                // first of this workgroup's rows, counted from begin
    bool real;
};

// s = 0: the rows in front of the first sequence, s = B + 1: those behind the last
__device__ __forceinline__ int pa_bound(const int* ends, int s, int B, int T) {
    if (s <= 0) return 0;
    if (s > B + 1) return T;
    const int e = ends[s - 1];
    return e < 0 ? 0 : e > T ? T : e;
}

__device__ __forceinline__ bool pa_find(const int* ends, int T, const int* ends2, int T2, int B, int slot, PaSeq& r) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 < B + 2; s0 += 64) {
        const int s = s0 + lane;
        const bool in = s < B + 2 && pa_bound(ends, s, B, T) / PA_ROWS + s <= slot;
        before += __popcll(__ballot(in));
    }
    const int s = __builtin_amdgcn_readfirstlane(before) - 1;
    if (s < 0) return false;
    r.begin = pa_bound(ends, s, B, T);
    const int end = pa_bound(ends, s + 1, B, T);
    r.n = end > r.begin ? end - r.begin : 0;
    r.row0 = (slot - (r.begin / PA_ROWS + s)) * PA_ROWS;
    r.real = s >= 1 && s <= B;
    r.begin2 = r.n2 = 0;
    if (r.real) {
        r.begin2 = pa_bound(ends2, s, B, T2);
        const int end2 = pa_bound(ends2, s + 1, B, T2);
        r.n2 = end2 > r.begin2 ? end2 - r.begin2 : 0;
    }
    r.begin = __builtin_amdgcn_readfirstlane(r.begin);
    r.n = __builtin_amdgcn_readfirstlane(r.n);
    r.begin2 = __builtin_amdgcn_readfirstlane(r.begin2);
    r.n2 = __builtin_amdgcn_readfirstlane(r.n2);
    r.row0 = __builtin_amdgcn_readfirstlane(r.row0);
    return r.row0 >= 0 && r.row0 < r.n;
}

// ---- tiles -------------------------------------------------------------------------------------------------------------------
template <int DHP> struct PaTile {
    static constexpr int RB = DHP * 2, CH = DHP / 8, PER = PA_TILE * CH / 256, BYTES = PA_TILE * RB;
    // the row-dependent xor on the index of a 16-byte piece: rows that share a 256-byte line of banks keep their order
    static __device__ __forceinline__ int swz(int row) { return (row / (256 / RB)) & (CH - 1); }
};

// byte offsets of the pieces that this thread moves of a tile; pieces past the head's width read as zeros (out of range of the buffer)
template <int DHP> __device__ __forceinline__ void pa_offsets(unsigned (&off)[PaTile<DHP>::PER], long long row_stride, int dh) {
    typedef PaTile<DHP> TL;
#pragma unroll
    for (int i = 0; i < TL::PER; ++i) {
        const int idx = i * 256 + (int)threadIdx.x, row = idx / TL::CH, c = idx % TL::CH;
        off[i] = c * 8 < dh ? (unsigned)(row * row_stride + c * 8) * 2u : 0xfffffff0u;
    }
}

// rows row0 ... row0 + 63 of a sequence's n rows that begin at base; rows past the end read as zeros
template <int DHP> __device__ __forceinline__ void pa_load(u32x4 (&st)[PaTile<DHP>::PER], const void* base, long long row_stride, int row0, int n, int dh,
                                                            const unsigned (&off)[PaTile<DHP>::PER]) {
    const int left = n - row0 < PA_TILE ? n - row0 : PA_TILE;
    const unsigned bytes = left > 0 ? (unsigned)((left - 1) * row_stride + dh) * 2u : 0u;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + row0 * row_stride * 2), 0, bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < PaTile<DHP>::PER; ++i) st[i] = __builtin_amdgcn_raw_buffer_load_b128(r, off[i], 0, 0);
}

template <int DHP> __device__ __forceinline__ void pa_store(char* lds, const u32x4 (&st)[PaTile<DHP>::PER]) {
    typedef PaTile<DHP> TL;
#pragma unroll
    for (int i = 0; i < TL::PER; ++i) {
        const int idx = i * 256 + (int)threadIdx.x, row = idx / TL::CH, c = idx % TL::CH;
        *(u32x4*)(lds + row * TL::RB + ((c ^ TL::swz(row)) << 4)) = st[i];
    }
}

// operand "row = tile row": lane's row, elements kc*16 + h*8 ... + 7
template <typename V8, int DHP> __device__ __forceinline__ V8 pa_row_frag(const char* lds, int row, int kc, int h) {
    typedef PaTile<DHP> TL;
    return *(const V8*)(lds + row * TL::RB + (((kc * 2 + h) ^ TL::swz(row)) << 4));
}

// operand "row = head dimension mt*32 + lane%32, contraction = the tile rows r0 + {0..3} + 4h and r0 + 8 + {0..3} + 4h": two transposed
// reads; within 16 lanes, lane i addresses row i/4, columns (i%4)*4 ... + 3 and receives column i of the four rows
template <typename V8, int DHP> __device__ __forceinline__ V8 pa_col_frag(const char* lds, int r0, int mt) {
    typedef PaTile<DHP> TL;
    const int lane = threadIdx.x & 63, li = lane & 15, row = r0 + 4 * (lane >> 5) + (li >> 2);
    const int col = mt * 32 + 16 * ((lane >> 4) & 1) + 4 * (li & 3);           // element column; its 16-byte piece is col / 8
    const char* p0 = lds + row * TL::RB + (((col >> 3) ^ TL::swz(row)) << 4) + (col & 7) * 2;
    const char* p1 = lds + (row + 8) * TL::RB + (((col >> 3) ^ TL::swz(row + 8)) << 4) + (col & 7) * 2;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(p0));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(p1));
    const s16x8 r = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(V8, r);
}

// this lane's owned row from global memory as operands; zeros past the head's width or for a row that does not exist
template <typename T, int DHP> __device__ __forceinline__ void pa_own(typename PaTypes<T>::v8 (&f)[DHP / 16], const PaView& x, long long row, int head, int dh, bool valid) {
    typedef typename PaTypes<T>::v8 v8;
    const T* p = (const T*)x.p + row * x.row + head * x.head;
#pragma unroll
    for (int kc = 0; kc < DHP / 16; ++kc) {
        const int d = kc * 16 + (int)((threadIdx.x >> 5) & 1) * 8;
        v8 z;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = (T)0.f;
        f[kc] = valid && d < dh ? *(const v8*)(p + d) : z;
    }
}

// a transposed result (rows = head dimensions, column = the lane's row) to memory
template <typename T, int DHP, typename F>
__device__ __forceinline__ void pa_put(const f32x16 (&acc)[DHP / 32], T* p, int dh, F&& f) {
    typedef typename PaTypes<T>::v4 v4;
#pragma unroll
    for (int mt = 0; mt < DHP / 32; ++mt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = mt * 32 + g * 8 + (int)((threadIdx.x >> 5) & 1) * 4;
            if (d < dh) {
                v4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (T)f(acc[mt][g * 4 + j]);
                *(v4*)(p + d) = w;
            }
        }
}

template <typename T> __device__ __forceinline__ typename PaTypes<T>::v8 pa_pack(const float* s) {
    typename PaTypes<T>::v8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)s[j];
    return r;
}

// ---- relative position bias ----------------------------------------------------------------------------------------------------
// LDS: the bias of every distance key - query in -far ... far for one head, in units of log2 like the scores.
__device__ __forceinline__ void pa_bias_fill(const PaArgs& a, int head, float* s_bias) {
    for (int i = threadIdx.x; i < 2 * a.far + 1; i += 256) {
        int b = a.bucket_of[i];
        b = b < 0 ? 0 : b >= a.buckets ? a.buckets - 1 : b;
        s_bias[i] = a.table[b * a.H + head] * 1.4426950408889634f;
    }
}
__device__ __forceinline__ int pa_clamp(int d, int far) { return d < -far ? -far : d > far ? far : d; }

// ================================================================================================================================
// forward
// ================================================================================================================================
template <typename T, int DHP, bool BIAS>
__global__ __launch_bounds__(256, 2) void pa_fwd_kernel(const PaArgs a) {
    typedef typename PaTypes<T>::v8 v8;
    typedef PaTile<DHP> TL;
    constexpr int KC = DHP / 16, MT = DHP / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // k, v tiles, two buffers of both; then the bias
    float* const s_bias = (float*)(smem + 4 * TL::BYTES);
    // heads that share k, v differ by Hk in their index: with workgroups dealt to the eight XCDs in turn, they meet in one L2
    const int hk = blockIdx.x % a.Hk, g = blockIdx.x / a.Hk % (a.H / a.Hk), head = hk * (a.H / a.Hk) + g;
    const int slot = a.slots - 1 - (int)(blockIdx.x / a.H);                // (ends of causal sequences, the longest rows, first)
    PaSeq sq;
    if (!pa_find(a.ends_q, a.Tq, a.ends_k, a.Tk, a.B, slot, sq)) return;
    if (!sq.real && !a.zero_rest) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
    const int w0 = sq.row0 + wave * 32, qi = w0 + col;                     // the wave's first row, the lane's row
    const bool qv = qi < sq.n;
    const int off = a.causal ? sq.n2 - sq.n : 0;                           // a causal row's last key is row + off
    if (BIAS) pa_bias_fill(a, head, s_bias);

    v8 bq[KC];
    pa_own<T, DHP>(bq, a.q, sq.begin + (qv ? qi : 0), head, a.dh, qv);
    f32x16 acc[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt] = pa_zero();
    float m = -INFINITY, l = 0.f;

    const int rows = sq.n - sq.row0 < PA_ROWS ? sq.n - sq.row0 : PA_ROWS;
    int keys = a.causal ? sq.row0 + rows + off : sq.n2;                    // keys that any row of the workgroup sees
    keys = keys < 0 ? 0 : keys < sq.n2 ? keys : sq.n2;
    const int tiles = (keys + PA_TILE - 1) / PA_TILE;
    const char* const kb = (const char*)a.k.p + (sq.begin2 * a.k.row + hk * a.k.head) * 2;
    const char* const vb = (const char*)a.v.p + (sq.begin2 * a.v.row + hk * a.v.head) * 2;
    unsigned ko[TL::PER], vo[TL::PER];
    pa_offsets<DHP>(ko, a.k.row, a.dh);
    pa_offsets<DHP>(vo, a.v.row, a.dh);
    u32x4 kst[TL::PER], vst[TL::PER];
    if (tiles > 0) {
        pa_load<DHP>(kst, kb, a.k.row, 0, sq.n2, a.dh, ko);
        pa_load<DHP>(vst, vb, a.v.row, 0, sq.n2, a.dh, vo);
        pa_store<DHP>(smem, kst);
        pa_store<DHP>(smem + TL::BYTES, vst);
    }
    __syncthreads();
    const int w_rows = sq.n - w0 < 32 ? sq.n - w0 : 32;                    // <= 0: the wave has no rows
    for (int t = 0; t < tiles; ++t) {
        const char* const lk = smem + (t & 1) * 2 * TL::BYTES;
        const char* const lv = lk + TL::BYTES;
        const int k0 = t * PA_TILE;
        if (t + 1 < tiles) {
            pa_load<DHP>(kst, kb, a.k.row, k0 + PA_TILE, sq.n2, a.dh, ko);
            pa_load<DHP>(vst, vb, a.v.row, k0 + PA_TILE, sq.n2, a.dh, vo);
        }
        if (w_rows > 0 && (!a.causal || k0 <= w0 + w_rows - 1 + off)) {
            f32x16 sc[2] = {pa_zero(), pa_zero()};
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) {
                sc[0] = pa_mfma(pa_row_frag<v8, DHP>(lk, col, kc, h), bq[kc], sc[0]);
                sc[1] = pa_mfma(pa_row_frag<v8, DHP>(lk, 32 + col, kc, h), bq[kc], sc[1]);
            }
            float s[32];
            const int dist0 = k0 + h * 4 - (qi + off);                     // distance of the lane's first score
            if (BIAS) {
                const int lo = k0 - (w0 + w_rows - 1 + off), hi = k0 + PA_TILE - 1 - (w0 + off);       // distances in the wave's tile
                if (hi <= -a.far || lo >= a.far) {
                    const float b = s_bias[hi <= -a.far ? 0 : 2 * a.far];
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[i] = sc[i >> 4][i & 15] * a.scale2 + b;
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        s[i] = sc[i >> 4][i & 15] * a.scale2 + s_bias[pa_clamp(dist0 + (i >> 2) * 8 + (i & 3), a.far) + a.far];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = sc[i >> 4][i & 15] * a.scale2;
            }
            if (k0 + PA_TILE > sq.n2 || (a.causal && k0 + PA_TILE - 1 > w0 + off)) {
                // key index - k0 of score i is (i >> 2) * 8 + h * 4 + (i & 3): beyond `last` it is not seen
                const int last = (a.causal && qi + off < sq.n2 - 1 ? qi + off : sq.n2 - 1) - k0 - h * 4;
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = (i >> 2) * 8 + (i & 3) <= last ? s[i] : -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int i = 1; i < 32; ++i) mx = fmaxf(mx, s[i]);
            mx = pa_half_max(mx);
            // The maximum moves only when a row's grows by more than 2^8: until then the old one keeps every term below 2^8, which
            // costs no precision, and the accumulators need no rescaling.
            if (__any(mx > m + 8.f)) {
                const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;       // (a row that has seen nothing yet stays at zero)
                const float alpha = __builtin_amdgcn_exp2f(m - ref);
                l *= alpha;
                m = mn;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[mt][i] *= alpha;
            }
            const float ref = m == -INFINITY ? 0.f : m;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                s[i] = __builtin_amdgcn_exp2f(s[i] - ref);
                sum += s[i];
            }
            l += sum;                                                      // (this half-wave's keys; joined at the end)
            // p is rounded to the type of v for the product (relative 2^-8 of each term in bf16, of either sign); the sum above is not.
            // Where the output feeds the bias's gradient, whose terms cancel, what that rounding leaves is multiplied as well.
            auto pv = [&](auto two) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const v8 p = pa_pack<T>(s + 8 * c);
                    v8 rest;
                    if constexpr (decltype(two)::value) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) rest[j] = (T)(s[8 * c + j] - (float)p[j]);
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const v8 f = pa_col_frag<v8, DHP>(lv, 16 * c, mt);
                        acc[mt] = pa_mfma(f, p, acc[mt]);
                        if constexpr (decltype(two)::value) acc[mt] = pa_mfma(f, rest, acc[mt]);
                    }
                }
            };
            if (BIAS && a.o32) pv(std::true_type());
            else pv(std::false_type());
        }
        if (t + 1 < tiles) {
            char* const nk = smem + ((t + 1) & 1) * 2 * TL::BYTES;
            pa_store<DHP>(nk, kst);
            pa_store<DHP>(nk + TL::BYTES, vst);
        }
        __syncthreads();
    }
    l = pa_half_sum(l);
    if (!qv) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const long long row = sq.begin + qi;
    pa_put<T, DHP>(acc, (T*)a.o.p + row * a.o.row + head * a.o.head, a.dh, [&](float x) { return x * inv; });
    if (a.o32) {
        float* const p = a.o32 + (row * a.H + head) * a.dh;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int d = mt * 32 + g4 * 8 + h * 4;
                if (d < a.dh) {
                    f32x4 w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = acc[mt][g4 * 4 + j] * inv;
                    *(f32x4*)(p + d) = w;
                }
            }
    }
    if (a.lse && h == 0) a.lse[(long long)head * a.Tq + row] = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
}

// ================================================================================================================================
// backward: dq (and D, and the bias's gradient); a wave owns 32 queries
// ================================================================================================================================
// The gradient of the bias is a sum of ds over equal distances first and over the distances of a bucket last.  Distances inside of
// (-far, far) are added up in LDS, one array per half-wave: the 32 lanes of a half hold 32 different distances of any one
// register, so that no two lanes of an instruction meet, and a wave's LDS operations are executed in order; what is beyond
// goes to two registers.  Every sum has a fixed order.  It is taken from the 32-bit ds, and D from the 32-bit output that the
// forward pass leaves for it, with p in two parts there (either rounding to 16 bits would be the largest error of such a sum,
// whose terms cancel: 5e-4 of the gradient instead of 1e-6).
template <typename T, int DHP, bool BIAS>
__global__ __launch_bounds__(256, 2) void pa_bwd_dq_kernel(const PaArgs a) {
    typedef typename PaTypes<T>::v8 v8;
    typedef PaTile<DHP> TL;
    constexpr int KC = DHP / 16, MT = DHP / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // k, v tiles, two buffers of both; then the bias and its sums
    const int width = 2 * a.far + 1;
    float* const s_bias = (float*)(smem + 4 * TL::BYTES);
    float* const s_sum = s_bias + width;                                   // [8][width]
    const int hk = blockIdx.x % a.Hk, g = blockIdx.x / a.Hk % (a.H / a.Hk), head = hk * (a.H / a.Hk) + g;
    const int slot = a.slots - 1 - (int)(blockIdx.x / a.H);
    const bool want_table = BIAS && a.dtable_part;
    float* const part = want_table ? a.dtable_part + ((long long)slot * a.H + head) * a.buckets : nullptr;
    PaSeq sq;
    if (!pa_find(a.ends_q, a.Tq, a.ends_k, a.Tk, a.B, slot, sq) || (!sq.real && !a.zero_rest)) {
        if (want_table)
            for (int i = threadIdx.x; i < a.buckets; i += 256) part[i] = 0.f;
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
    const int w0 = sq.row0 + wave * 32, qi = w0 + col;
    const bool qv = qi < sq.n;
    const int off = a.causal ? sq.n2 - sq.n : 0;
    const long long row = sq.begin + (qv ? qi : 0);
    if (BIAS) {
        pa_bias_fill(a, head, s_bias);
        if (want_table)
            for (int i = threadIdx.x; i < 8 * width; i += 256) s_sum[i] = 0.f;
    }
    float* const my_sum = s_sum + (threadIdx.x >> 5) * width;
    float before = 0.f, after = 0.f;                                       // ds at distances <= -far, >= far

    v8 bq[KC], bdo[KC];
    pa_own<T, DHP>(bq, a.q, row, head, a.dh, qv);
    pa_own<T, DHP>(bdo, a.dout, row, head, a.dh, qv);
    float dsum = 0.f;
    if (a.o32) {
        const float* const o = a.o32 + (row * a.H + head) * a.dh;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            const int d = kc * 16 + h * 8;
            if (d < a.dh) {
                const f32x4 lo = *(const f32x4*)(o + d), hi = *(const f32x4*)(o + d + 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) dsum += (float)bdo[kc][j] * lo[j];
#pragma unroll
                for (int j = 0; j < 4; ++j) dsum += (float)bdo[kc][4 + j] * hi[j];
            }
        }
    } else {
        v8 of[KC];
        pa_own<T, DHP>(of, a.o, row, head, a.dh, qv);
#pragma unroll
        for (int kc = 0; kc < KC; ++kc)
#pragma unroll
            for (int j = 0; j < 8; ++j) dsum += (float)bdo[kc][j] * (float)of[kc][j];
    }
    dsum = pa_half_sum(dsum);
    const float lse = qv ? a.lse[(long long)head * a.Tq + row] : 0.f;
    if (qv && h == 0) a.dsum[(long long)head * a.Tq + row] = dsum;
    f32x16 acc[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt] = pa_zero();

    const int rows = sq.n - sq.row0 < PA_ROWS ? sq.n - sq.row0 : PA_ROWS;
    int keys = a.causal ? sq.row0 + rows + off : sq.n2;
    keys = keys < 0 ? 0 : keys < sq.n2 ? keys : sq.n2;
    const int tiles = (keys + PA_TILE - 1) / PA_TILE;
    const char* const kb = (const char*)a.k.p + (sq.begin2 * a.k.row + hk * a.k.head) * 2;
    const char* const vb = (const char*)a.v.p + (sq.begin2 * a.v.row + hk * a.v.head) * 2;
    unsigned ko[TL::PER], vo[TL::PER];
    pa_offsets<DHP>(ko, a.k.row, a.dh);
    pa_offsets<DHP>(vo, a.v.row, a.dh);
    u32x4 kst[TL::PER], vst[TL::PER];
    if (tiles > 0) {
        pa_load<DHP>(kst, kb, a.k.row, 0, sq.n2, a.dh, ko);
        pa_load<DHP>(vst, vb, a.v.row, 0, sq.n2, a.dh, vo);
        pa_store<DHP>(smem, kst);
        pa_store<DHP>(smem + TL::BYTES, vst);
    }
    __syncthreads();
    const int w_rows = sq.n - w0 < 32 ? sq.n - w0 : 32;
    for (int t = 0; t < tiles; ++t) {
        const char* const lk = smem + (t & 1) * 2 * TL::BYTES;
        const char* const lv = lk + TL::BYTES;
        if (t + 1 < tiles) {
            pa_load<DHP>(kst, kb, a.k.row, (t + 1) * PA_TILE, sq.n2, a.dh, ko);
            pa_load<DHP>(vst, vb, a.v.row, (t + 1) * PA_TILE, sq.n2, a.dh, vo);
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int k0 = t * PA_TILE + sub * 32;
            if (w_rows > 0 && k0 < sq.n2 && (!a.causal || k0 <= w0 + w_rows - 1 + off)) {
                f32x16 sc = pa_zero(), dp = pa_zero();
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    sc = pa_mfma(pa_row_frag<v8, DHP>(lk, sub * 32 + col, kc, h), bq[kc], sc);
                    dp = pa_mfma(pa_row_frag<v8, DHP>(lv, sub * 32 + col, kc, h), bdo[kc], dp);
                }
                float ds[16];
                const int dist0 = k0 + h * 4 - (qi + off);
                const int lo = k0 - (w0 + w_rows - 1 + off), hi = k0 + 31 - (w0 + off);
                const bool far = BIAS && (hi <= -a.far || lo >= a.far);
                if (BIAS && !far) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        ds[i] = __builtin_amdgcn_exp2f(sc[i] * a.scale2 + (s_bias[pa_clamp(dist0 + (i >> 2) * 8 + (i & 3), a.far) + a.far] - lse));
                } else {
                    const float b = BIAS ? s_bias[hi <= -a.far ? 0 : 2 * a.far] - lse : -lse;
#pragma unroll
                    for (int i = 0; i < 16; ++i) ds[i] = __builtin_amdgcn_exp2f(sc[i] * a.scale2 + b);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[i] *= dp[i] - dsum;
                if (k0 + 32 > sq.n2 || w_rows < 32 || (a.causal && k0 + 31 > w0 + off)) {
                    int last = (a.causal && qi + off < sq.n2 - 1 ? qi + off : sq.n2 - 1) - k0 - h * 4;
                    if (!qv) last = -1;
#pragma unroll
                    for (int i = 0; i < 16; ++i) ds[i] = (i >> 2) * 8 + (i & 3) <= last ? ds[i] : 0.f;
                }
                if (want_table) {
                    if (far) {
                        float sum = 0.f;
#pragma unroll
                        for (int i = 0; i < 16; ++i) sum += ds[i];
                        if (hi <= -a.far) before += sum;
                        else after += sum;
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int d = dist0 + (i >> 2) * 8 + (i & 3);
                            if (d <= -a.far) before += ds[i];
                            else if (d >= a.far) after += ds[i];
                            else __hip_atomic_fetch_add(my_sum + d + a.far, ds[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                        }
                    }
                }
                // ds is rounded to the type of k for the product (see p in the forward pass)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const v8 p = pa_pack<T>(ds + 8 * c);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) acc[mt] = pa_mfma(pa_col_frag<v8, DHP>(lk, sub * 32 + 16 * c, mt), p, acc[mt]);
                }
            }
        }
        if (t + 1 < tiles) {
            char* const nk = smem + ((t + 1) & 1) * 2 * TL::BYTES;
            pa_store<DHP>(nk, kst);
            pa_store<DHP>(nk + TL::BYTES, vst);
        }
        __syncthreads();
    }
    if (qv) pa_put<T, DHP>(acc, (T*)a.dq.p + row * a.dq.row + head * a.dq.head, a.dh, [&](float x) { return x * a.scale; });
    if (!want_table) return;
    before = wave_sum(before);
    after = wave_sum(after);
    if (lane == 0) { s_bias[wave * 2] = before; s_bias[wave * 2 + 1] = after; }       // (the bias itself is no longer needed; width >= 9)
    __syncthreads();
    for (int i = threadIdx.x; i < width; i += 256) {
        float x = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) x += s_sum[k * width + i];
        if (i == 0) x += (s_bias[0] + s_bias[2]) + (s_bias[4] + s_bias[6]);
        if (i == 2 * a.far) x += (s_bias[1] + s_bias[3]) + (s_bias[5] + s_bias[7]);
        s_sum[i] = x;                                  // (only this thread reads or writes column i)
    }
    __syncthreads();
    for (int b = threadIdx.x; b < a.buckets; b += 256) {
        float x = 0.f;
        for (int i = 0; i < width; ++i) {
            int k = a.bucket_of[i];
            k = k < 0 ? 0 : k >= a.buckets ? a.buckets - 1 : k;
            x += k == b ? s_sum[i] : 0.f;
        }
        part[b] = x;
    }
}

// dtable[b][head] = sum over the slots, in order, in 64 bits; one workgroup per head
__global__ __launch_bounds__(256) void pa_dtable_kernel(const float* __restrict__ part, int slots, int H, int buckets, float* __restrict__ dtable) {
    const int head = blockIdx.x;
    for (int b = threadIdx.x; b < buckets; b += 256) {
        double x = 0.0;
#pragma unroll 8
        for (int s = 0; s < slots; ++s) x += (double)part[((long long)s * H + head) * buckets + b];
        dtable[(long long)b * H + head] = (float)x;
    }
}

// ================================================================================================================================
// backward: dk, dv; a wave owns 32 keys and walks over the queries of every head that shares them
// ================================================================================================================================
template <typename T, int DHP, bool BIAS>
__global__ __launch_bounds__(256, DHP > 64 ? 1 : 2) void pa_bwd_dkv_kernel(const PaArgs a) {
    typedef typename PaTypes<T>::v8 v8;
    typedef PaTile<DHP> TL;
    constexpr int KC = DHP / 16, MT = DHP / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // q, do tiles, two buffers of both; lse and D of their rows; the bias
    float* const s_row = (float*)(smem + 4 * TL::BYTES);                   // [2][2][64]
    float* const s_bias = s_row + 4 * PA_TILE;
    const int hk = blockIdx.x % a.Hk, group = a.H / a.Hk;
    const int slot = (int)(blockIdx.x / a.Hk);                             // (starts of causal sequences, the most queries, first)
    PaSeq sq;                                                              // begin, n: keys; begin2, n2: queries
    if (!pa_find(a.ends_k, a.Tk, a.ends_q, a.Tq, a.B, slot, sq)) return;
    if (!sq.real && !a.zero_rest) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
    const int w0 = sq.row0 + wave * 32, ki = w0 + col;
    const bool kv = ki < sq.n;
    const int off = a.causal ? sq.n - sq.n2 : 0;
    const long long row = sq.begin + (kv ? ki : 0);
    v8 bk[KC], bv[KC];
    pa_own<T, DHP>(bk, a.k, row, hk, a.dh, kv);
    pa_own<T, DHP>(bv, a.v, row, hk, a.dh, kv);
    f32x16 dk[MT], dv[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) { dk[mt] = pa_zero(); dv[mt] = pa_zero(); }
    int first = a.causal ? sq.row0 - off : 0;                              // the first query that sees any key of the workgroup
    first = first < 0 ? 0 : first / PA_TILE * PA_TILE;
    const int tiles = sq.n2 > first ? (sq.n2 - first + PA_TILE - 1) / PA_TILE : 0, steps = tiles * group;
    unsigned qo[TL::PER], po[TL::PER];
    pa_offsets<DHP>(qo, a.q.row, a.dh);
    pa_offsets<DHP>(po, a.dout.row, a.dh);
    u32x4 qst[TL::PER], pst[TL::PER];
    float rst = 0.f;                                                       // threads 0 .. 63: lse of a query, 64 .. 127: its D
    auto fetch = [&](int step) {
        const int hd = hk * group + step / tiles, q0 = first + step % tiles * PA_TILE;
        pa_load<DHP>(qst, (const char*)a.q.p + (sq.begin2 * a.q.row + hd * a.q.head) * 2, a.q.row, q0, sq.n2, a.dh, qo);
        pa_load<DHP>(pst, (const char*)a.dout.p + (sq.begin2 * a.dout.row + hd * a.dout.head) * 2, a.dout.row, q0, sq.n2, a.dh, po);
        if (threadIdx.x < 2 * PA_TILE) {
            const int q = q0 + (threadIdx.x & (PA_TILE - 1));
            const long long at = (long long)hd * a.Tq + sq.begin2 + q;
            if (threadIdx.x < PA_TILE) {
                rst = q < sq.n2 ? a.lse[at] : INFINITY;
                if (rst == -INFINITY) rst = INFINITY;                      // no key seen, or no query: every probability comes out as zero
            } else
                rst = q < sq.n2 ? a.dsum[at] : 0.f;
        }
    };
    auto keep = [&](int buf) {
        char* const p = smem + buf * 2 * TL::BYTES;
        pa_store<DHP>(p, qst);
        pa_store<DHP>(p + TL::BYTES, pst);
        if (threadIdx.x < 2 * PA_TILE) s_row[buf * 2 * PA_TILE + threadIdx.x] = rst;
    };
    if (steps > 0) {
        fetch(0);
        keep(0);
    }
    const int w_rows = sq.n - w0 < 32 ? sq.n - w0 : 32;
    for (int step = 0; step < steps; ++step) {
        if (BIAS && step % tiles == 0) {
            __syncthreads();
            pa_bias_fill(a, hk * group + step / tiles, s_bias);
        }
        __syncthreads();
        const char* const lq = smem + (step & 1) * 2 * TL::BYTES;
        const char* const lp = lq + TL::BYTES;
        const float* const lr = s_row + (step & 1) * 2 * PA_TILE;
        if (step + 1 < steps) fetch(step + 1);
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int q0 = first + step % tiles * PA_TILE + sub * 32;
            if (w_rows > 0 && q0 < sq.n2 && (!a.causal || q0 + 31 + off >= w0)) {
                f32x16 sc = pa_zero(), dp = pa_zero();
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    sc = pa_mfma(pa_row_frag<v8, DHP>(lq, sub * 32 + col, kc, h), bk[kc], sc);
                    dp = pa_mfma(pa_row_frag<v8, DHP>(lp, sub * 32 + col, kc, h), bv[kc], dp);
                }
                float p[16], ds[16];
                const int dist0 = ki - (q0 + h * 4 + off);                 // distance of the lane's first score; later rows are nearer
                float bc = 0.f;
                bool far = true;
                if (BIAS) {
                    const int lo = w0 - (q0 + 31 + off), hi = w0 + w_rows - 1 - (q0 + off);
                    far = hi <= -a.far || lo >= a.far;
                    if (far) bc = s_bias[hi <= -a.far ? 0 : 2 * a.far];
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 ls = *(const f32x4*)(lr + sub * 32 + g * 8 + h * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int i = g * 4 + j;
                        const float b = BIAS && !far ? s_bias[pa_clamp(dist0 - g * 8 - j, a.far) + a.far] : bc;
                        p[i] = __builtin_amdgcn_exp2f(sc[i] * a.scale2 + (b - ls[j]));
                    }
                }
                if (a.causal && w0 + w_rows - 1 > q0 + off) {
                    const int firstq = ki - off - q0 - h * 4;              // query index of a row that sees this key
#pragma unroll
                    for (int i = 0; i < 16; ++i) p[i] = (i >> 2) * 8 + (i & 3) >= firstq ? p[i] : 0.f;
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const v8 pp = pa_pack<T>(p + 8 * c);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) dv[mt] = pa_mfma(pa_col_frag<v8, DHP>(lp, sub * 32 + 16 * c, mt), pp, dv[mt]);
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 dd = *(const f32x4*)(lr + PA_TILE + sub * 32 + g * 8 + h * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) ds[g * 4 + j] = p[g * 4 + j] * (dp[g * 4 + j] - dd[j]);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const v8 pp = pa_pack<T>(ds + 8 * c);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) dk[mt] = pa_mfma(pa_col_frag<v8, DHP>(lq, sub * 32 + 16 * c, mt), pp, dk[mt]);
                }
            }
        }
        if (step + 1 < steps) keep((step + 1) & 1);
    }
    if (!kv) return;
    pa_put<T, DHP>(dk, (T*)a.dk.p + row * a.dk.row + hk * a.dk.head, a.dh, [&](float x) { return x * a.scale; });
    pa_put<T, DHP>(dv, (T*)a.dv.p + row * a.dv.row + hk * a.dv.head, a.dh, [&](float x) { return x; });
}

// ================================================================================================================================
// launch
// ================================================================================================================================
namespace {
constexpr int PA_MAX_FAR = 1024;

int pa_launch(void (*kernel)(const PaArgs), unsigned grid, size_t lds, const PaArgs& a, hipStream_t st) {
    if (lds > 64 * 1024 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) {
        ddpm_set_error("packed_attention: cannot reserve %zu bytes of LDS", lds);
        return DDPM_EHIP;
    }
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), lds, st, a);
    return ddpm_check_launch("packed_attention");
}

template <typename T, int DHP, bool BIAS>
int pa_launch_fwd(const PaArgs& a, hipStream_t st) {
    return pa_launch(pa_fwd_kernel<T, DHP, BIAS>, (unsigned)(a.slots * a.H), 4 * PaTile<DHP>::BYTES + (BIAS ? (2 * a.far + 1) * 4 : 0), a, st);
}

template <typename T, int DHP, bool BIAS>
int pa_launch_bwd(PaArgs a, float* dtable, hipStream_t st) {
    const size_t width = (2 * a.far + 1) * 4;
    if (a.Tq > 0) {
        if (const int rc = pa_launch(pa_bwd_dq_kernel<T, DHP, BIAS>, (unsigned)(a.slots * a.H), 4 * PaTile<DHP>::BYTES + (BIAS ? (a.dtable_part ? 9 : 1) * width : 0), a, st)) return rc;
    }
    if (a.dtable_part)
        hipLaunchKernelGGL(pa_dtable_kernel, dim3((unsigned)a.H), dim3(256), 0, st, a.dtable_part, a.Tq > 0 ? a.slots : 0, a.H, a.buckets, dtable);
    a.slots = a.Tk / PA_ROWS + a.B + 2;
    if (a.Tk == 0) return ddpm_check_launch("packed_attention_backward");
    return pa_launch(pa_bwd_dkv_kernel<T, DHP, BIAS>, (unsigned)(a.slots * a.Hk), 4 * PaTile<DHP>::BYTES + 16 * PA_TILE + (BIAS ? width : 0), a, st);
}

template <typename F> int pa_dispatch(const ddpm_packed_attn_desc* d, F&& f) {
    const int pad = d->dh <= 32 ? 32 : d->dh <= 64 ? 64 : 128;
#define PA_CASE(T, DHP) (d->table ? f(T(), std::integral_constant<int, DHP>(), std::true_type()) : f(T(), std::integral_constant<int, DHP>(), std::false_type()))
    if (d->dtype == DDPM_BF16) return pad == 32 ? PA_CASE(bf16, 32) : pad == 64 ? PA_CASE(bf16, 64) : PA_CASE(bf16, 128);
    return pad == 32 ? PA_CASE(f16, 32) : pad == 64 ? PA_CASE(f16, 64) : PA_CASE(f16, 128);
#undef PA_CASE
}

int pa_view(const char* name, const void* p, int64_t row, int64_t head, int rows, int heads, int dh, PaView& v) {
    v = {(void*)p, row, head};
    if (rows == 0) return DDPM_OK;
    DDPM_REQUIRE(p && (uintptr_t)p % 16 == 0, "packed_attention: %s is null or not 16-byte aligned", name);
    DDPM_REQUIRE((rows == 1 || (row % 8 == 0 && row > 0)) && (heads == 1 || (head % 8 == 0 && head > 0)), "packed_attention: strides of %s (%lld, %lld) must be positive multiples of 8",
                 name, (long long)row, (long long)head);
    DDPM_REQUIRE(rows == 1 || row < (1 << 24), "packed_attention: rows of %s are %lld elements apart (at most 2^24 - 1)", name, (long long)row);
    DDPM_REQUIRE((heads == 1 || head >= dh) && (rows == 1 || row >= dh), "packed_attention: strides of %s are shorter than a head", name);
    return DDPM_OK;
}

int pa_setup(const ddpm_packed_attn_desc* d, bool bwd, PaArgs& a) {
    DDPM_REQUIRE(d, "packed_attention: null descriptor");
    DDPM_REQUIRE(d->dtype == DDPM_BF16 || d->dtype == DDPM_F16, "packed_attention: element type %d (bf16 or fp16)", d->dtype);
    DDPM_REQUIRE(d->dh >= 8 && d->dh <= 128 && d->dh % 8 == 0, "packed_attention: head width %d (a multiple of 8 up to 128)", d->dh);
    DDPM_REQUIRE(d->H >= 1 && d->Hk >= 1 && d->H % d->Hk == 0 && d->H <= 65535, "packed_attention: %d heads over %d shared ones", d->H, d->Hk);
    DDPM_REQUIRE(d->Tq >= 0 && d->Tk >= 0 && d->B >= 0 && d->Tq < (1 << 30) && d->Tk < (1 << 30) && d->B < (1 << 24), "packed_attention: %d queries, %d keys, %d sequences", d->Tq, d->Tk, d->B);
    DDPM_REQUIRE(d->ends_q && d->ends_k, "packed_attention: the sequences' boundaries are missing");
    DDPM_REQUIRE(d->scale > 0.f && d->scale < INFINITY, "packed_attention: scale must be positive and finite");
    DDPM_REQUIRE((int64_t)(d->Tq / PA_ROWS + d->B + 2) * d->H < (1ll << 31) && (int64_t)(d->Tk / PA_ROWS + d->B + 2) * d->Hk < (1ll << 31), "packed_attention: too many workgroups");
    DDPM_REQUIRE(!d->table == !d->bucket_of, "packed_attention: the bias needs both its table and the buckets of the distances");
    a = {};
    if (d->table) {
        DDPM_REQUIRE(d->far >= 4 && d->far <= PA_MAX_FAR, "packed_attention: distances to %d (4 to %d)", d->far, PA_MAX_FAR);
        DDPM_REQUIRE(d->buckets >= 1 && d->buckets <= 65536, "packed_attention: %d buckets", d->buckets);
    } else
        DDPM_REQUIRE(!d->dtable, "packed_attention: a gradient of a bias that is not there");
    if (const int rc = pa_view("q", d->q, d->q_row, d->q_head, d->Tq, d->H, d->dh, a.q)) return rc;
    if (const int rc = pa_view("k", d->k, d->k_row, d->k_head, d->Tk, d->Hk, d->dh, a.k)) return rc;
    if (const int rc = pa_view("v", d->v, d->v_row, d->v_head, d->Tk, d->Hk, d->dh, a.v)) return rc;
    if (const int rc = pa_view("o", d->o, d->o_row, d->o_head, d->Tq, d->H, d->dh, a.o)) return rc;
    if (bwd) {
        if (const int rc = pa_view("dout", d->dout, d->dout_row, d->dout_head, d->Tq, d->H, d->dh, a.dout)) return rc;
        if (const int rc = pa_view("dq", d->dq, d->dq_row, d->dq_head, d->Tq, d->H, d->dh, a.dq)) return rc;
        if (const int rc = pa_view("dk", d->dk, d->dk_row, d->dk_head, d->Tk, d->Hk, d->dh, a.dk)) return rc;
        if (const int rc = pa_view("dv", d->dv, d->dv_row, d->dv_head, d->Tk, d->Hk, d->dh, a.dv)) return rc;
        DDPM_REQUIRE(d->Tq == 0 || (d->lse && d->dsum), "packed_attention: backward needs lse and the workspace dsum");
        DDPM_REQUIRE(!d->dtable || d->dtable_part, "packed_attention: the bias's gradient needs the workspace dtable_part");
    }
    a.o32 = d->o32; a.lse = d->lse; a.dsum = d->dsum;
    a.ends_q = d->ends_q; a.ends_k = d->ends_k;
    a.table = d->table; a.bucket_of = d->bucket_of; a.buckets = d->buckets; a.far = d->table ? d->far : 0;
    a.dtable_part = bwd && d->dtable ? d->dtable_part : nullptr;
    a.Tq = d->Tq; a.Tk = d->Tk; a.B = d->B; a.H = d->H; a.Hk = d->Hk; a.dh = d->dh; a.causal = d->causal; a.zero_rest = d->zero_rest;
    a.slots = d->Tq / PA_ROWS + d->B + 2;
    a.scale = d->scale;
    a.scale2 = d->scale * 1.4426950408889634f;
    return DDPM_OK;
}
}  // namespace

extern "C" int ddpm_packed_attn_slots(int Tq, int B) { return Tq / PA_ROWS + B + 2; }

extern "C" int ddpm_packed_attention_forward(const ddpm_packed_attn_desc* d, ddpm_stream_t stream) {
    PaArgs a;
    if (const int rc = pa_setup(d, false, a)) return rc;
    if (d->Tq == 0) return DDPM_OK;
    return pa_dispatch(d, [&](auto t, auto pad, auto bias) { return pa_launch_fwd<decltype(t), decltype(pad)::value, decltype(bias)::value>(a, (hipStream_t)stream); });
}

extern "C" int ddpm_packed_attention_backward(const ddpm_packed_attn_desc* d, ddpm_stream_t stream) {
    PaArgs a;
    if (const int rc = pa_setup(d, true, a)) return rc;
    return pa_dispatch(d, [&](auto t, auto pad, auto bias) { return pa_launch_bwd<decltype(t), decltype(pad)::value, decltype(bias)::value>(a, d->dtable, (hipStream_t)stream); });
}
