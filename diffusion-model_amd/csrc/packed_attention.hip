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
// Sequences.  The launch has one slot for every 128 rows plus one per sequence, which is enough whatever the lengths are; the host does not know
// them.  A workgroup finds its sequence from the boundaries, a lane to each.  Rows outside of all sequences are two more sequences without keys: their results are zeros where the caller wants that, and they are not touched otherwise.
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
    float* dkv_part;                         // [2][splits][Tk][Hk][dh], where the queries of a key are split over workgroups
    int buckets, far;
    int Tq, Tk, B, H, Hk, dh, causal, zero_rest, slots, splits;
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

// A wave's LDS operations are executed in order; the compiler keeps to it here, where lanes read what others wrote
__device__ __forceinline__ void pa_wave_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// Order of N products and their operands' LDS reads (READS each) in what the compiler schedules together: the first AHEAD products' reads in
// front, then one product's at a time, so that a read has AHEAD products to arrive in
template <int N, int READS, int AHEAD> __device__ __forceinline__ void pa_order() {
    constexpr int A = AHEAD < N ? AHEAD : N;
    __builtin_amdgcn_sched_group_barrier(0x100, A * READS, 0);
#pragma unroll
    for (int i = 0; i < N - A; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, A, 0);
}

// ---- sequences ---------------------------------------------------------------------------------------------------------------
struct PaSeq {
    int begin, n;            // rows of the side that the launch's slots run over
    int begin2, n2;          // rows of the other side
    int row0;                // first of this workgroup's rows, counted from begin
};

// s = 0: the rows in front of the first sequence, s = B + 1: those behind the last
__device__ __forceinline__ int pa_bound(const int* ends, int s, int B, int T) {
    if (s <= 0) return 0;
    if (s > B + 1) return T;
    const int e = ends[s - 1];
    return e < 0 ? 0 : e > T ? T : e;
}

// sum over the lanes up to and including this one, without a trip through LDS (data-parallel moves within rows of 16, then across)
__device__ __forceinline__ int pa_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);        // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);        // the last of rows 0 and 2 to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);        // the last of row 1 to rows 2 and 3
    return v;
}

// The workgroup's rows: `rank` counts the tiles of 128 rows of all sequences, those with the most of the other side's rows first, so that the
// longest workgroups begin first and short ones fill the end (against the order by slots below, in a row of calls: training batch of 2048 ... 1 causal
// tokens, forward 108 -> 95 us, backward 360 -> 320; eight of 2048, backward 644 -> 558; but 8192 + 7937 tokens, backward 3.60 -> 3.70 ms).  A lane holds a sequence; the level that the rank falls into is found by bisection: causal, the tile's index within its sequence
// (queries: a later one sees more keys) or its distance from the end (keys: an earlier one is seen by more queries); otherwise the other
// side's length in tiles.  More sequences than lanes: by slots, in order.
template <bool KEYS>
__device__ __forceinline__ bool pa_find(const int* ends, int T, const int* ends2, int T2, int B, int zero_rest, int causal, int rank, int slots, PaSeq& r) {
    const int lane = threadIdx.x & 63;
    if (B + 2 <= 64) {
        const bool real = lane >= 1 && lane <= B;
        const int begin = pa_bound(ends, lane, B, T), end = lane < B + 2 ? pa_bound(ends, lane + 1, B, T) : begin;
        const int begin2 = pa_bound(ends2, lane, B, T2), end2 = real ? pa_bound(ends2, lane + 1, B, T2) : begin2;
        const int tiles = end > begin && (real || zero_rest) ? (end - begin + PA_ROWS - 1) / PA_ROWS : 0;
        const int tiles2 = end2 > begin2 ? (end2 - begin2 + PA_TILE - 1) / PA_TILE : 0;
        auto beyond = [&](int level) {                                     // tiles at this level and above
            return __builtin_amdgcn_readlane(pa_scan(causal ? (tiles > level ? tiles - level : 0) : tiles2 >= level ? tiles : 0), 63);
        };
        if (beyond(0) <= rank) return false;
        int level = 0, above = 0;
        for (int bit = 1 << (31 - __builtin_clz(causal ? T / PA_ROWS + 1 : T2 / PA_TILE + 1)); bit > 0; bit >>= 1) {
            const int n = beyond(level + bit);
            if (n > rank) level += bit;
            else above = n;                                                // (of the lowest level tried that is too high: level + 1 in the end)
        }
        // the tiles of just this level, sequence by sequence
        const int here = causal ? tiles > level : tiles2 == level ? tiles : 0;
        const int upto = pa_scan(here), at = rank - above, s = __ffsll(__ballot(upto > at)) - 1;
        const int of = __builtin_amdgcn_readlane(tiles, s), within = at - (__builtin_amdgcn_readlane(upto, s) - __builtin_amdgcn_readlane(here, s));
        r.begin = __builtin_amdgcn_readlane(begin, s);
        r.n = __builtin_amdgcn_readlane(end, s) - r.begin;
        r.begin2 = __builtin_amdgcn_readlane(begin2, s);
        r.n2 = __builtin_amdgcn_readlane(end2, s) - r.begin2;
        r.n2 = r.n2 > 0 ? r.n2 : 0;
        r.row0 = (causal ? (KEYS ? of - 1 - level : level) : within) * PA_ROWS;
        return true;
    }
    const int slot = KEYS ? rank : slots - 1 - rank;
    int before = 0;
    for (int s0 = 0; s0 < B + 2; s0 += 64)
        before += __popcll(__ballot(s0 + lane < B + 2 && pa_bound(ends, s0 + lane, B, T) / PA_ROWS + s0 + lane <= slot));
    const int s = __builtin_amdgcn_readfirstlane(before) - 1;
    if (s < 0) return false;
    const bool real = s >= 1 && s <= B;
    r.begin = __builtin_amdgcn_readfirstlane(pa_bound(ends, s, B, T));
    r.n = __builtin_amdgcn_readfirstlane(pa_bound(ends, s + 1, B, T)) - r.begin;
    r.row0 = (slot - (r.begin / PA_ROWS + s)) * PA_ROWS;
    r.begin2 = __builtin_amdgcn_readfirstlane(pa_bound(ends2, s, B, T2));
    r.n2 = real ? __builtin_amdgcn_readfirstlane(pa_bound(ends2, s + 1, B, T2)) - r.begin2 : 0;
    r.n2 = r.n2 > 0 ? r.n2 : 0;
    return r.row0 >= 0 && r.row0 < r.n && (real || zero_rest);
}

// ---- tiles -------------------------------------------------------------------------------------------------------------------
template <int DHP, int ROWS = PA_TILE> struct PaTile {
    static constexpr int RB = DHP * 2, CH = DHP / 8, BYTES = ROWS * RB;
    static constexpr int PER = 1024 / RB, ROUNDS = ROWS / (4 * PER);       // rows that a wave's load fills, loads of each of the four waves
    // The row-dependent xor on the index of a 16-byte piece.  Reads along rows: the same piece of 16 consecutive rows lies on 16 different
    // places of the 256-byte line of banks.  Transposed reads: 64 bytes each of four consecutive rows lie on its four quarters.
    static __device__ __forceinline__ int swz(int row) {
        if constexpr (CH == 16) return (row & 3) << 2 | (row >> 2 & 3);
        else if constexpr (CH == 8) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
        else return row >> 2 & 3;
    }
};

// Tiles go from memory to LDS without passing through registers (buffer_load ... lds: lane i's 16 bytes to m0 + 16 i), which leaves those to
// operands in flight.  The lane's piece of its wave's first load as a byte offset: the place in LDS decides which piece it is.  Rows past
// the end and pieces past the head's width are out of the buffer's range and arrive as zeros.
template <int DHP> __device__ __forceinline__ unsigned pa_piece(long long row_stride, int dh) {
    typedef PaTile<DHP> TL;
    const int lane = threadIdx.x & 63, row = (threadIdx.x >> 6) * TL::PER + lane / TL::CH, c = (lane % TL::CH) ^ TL::swz(row);
    return c * 8 < dh ? (unsigned)(row * row_stride + c * 8) * 2u : 0xfffffff0u;
}
#pragma clang diagnostic ignored "-Winline-asm"        /* (m0 is named as changed below; nothing keeps a value in it) */
// Rows row0 ... row0 + ROWS - 1 of a sequence's n rows that begin at base, to LDS at `lds`.  In assembly, since the compiler would wait for
// such a load before the next read of any LDS: pa_arrived() is the wait.
template <int DHP, int ROWS> __device__ __forceinline__ void pa_load(unsigned lds, const void* base, long long row_stride, int row0, int n, int dh, unsigned piece) {
    typedef PaTile<DHP, ROWS> TL;
    const int left = n - row0 < ROWS ? n - row0 : ROWS;
    const unsigned bytes = left > 0 ? (unsigned)((left - 1) * row_stride + dh) * 2u : 0u;
    const unsigned long long at = (unsigned long long)((const char*)base + row0 * row_stride * 2);
    const u32x4 buffer = {(unsigned)__builtin_amdgcn_readfirstlane((unsigned)at), (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(at >> 32)),
                          (unsigned)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
    const unsigned to = __builtin_amdgcn_readfirstlane(lds + (threadIdx.x >> 6) * 1024u);
#pragma unroll
    for (int i = 0; i < TL::ROUNDS; ++i)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                     :: "s"(to + i * 4096u), "v"(piece), "s"(buffer), "s"((unsigned)(i * 4 * TL::PER * row_stride) * 2u) : "memory", "m0");
}
// Every load of this wave has arrived (vmcnt 0); the barrier behind it says so for all waves.  As a builtin, so that the compiler knows of it: its own
// wait for loads in front of the loop would otherwise stand inside, behind the next tile's loads.
__device__ __forceinline__ void pa_arrived() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ unsigned pa_lds(const char* p) { return (unsigned)(unsigned long long)(const __attribute__((address_space(3))) char*)p; }

// Operands from a tile.  A lane's place in it is a number per kind of read; the xor moves only bits below a row, so that the 16-byte
// pieces of a row, and the columns of a transposed read, are that number with a constant xored in, and everything else is an
// immediate offset.  pa_opaque, once per tile, keeps the compiler from computing all of those in advance: for heads of 128 they would take
// two dozen registers that it then keeps in scratch memory.
//   "row = tile row": the lane's row, elements kc*16 + h*8 ... + 7
template <int DHP> __device__ __forceinline__ unsigned pa_row_place(int row, int h) {
    typedef PaTile<DHP> TL;
    return row * TL::RB + ((h ^ TL::swz(row)) << 4);
}
template <typename V8, int DHP> __device__ __forceinline__ V8 pa_row_frag(const char* lds, unsigned place, int kc) { return *(const V8*)(lds + (place ^ (kc << 5))); }
//   "row = head dimension mt*32 + lane%32, contraction = the tile rows r0 + {0..3} + 4h and r0 + 8 + {0..3} + 4h" (r0 a multiple of 16): two
// transposed reads; within 16 lanes, lane i addresses row i/4, columns (i%4)*4 ... + 3 and receives column i of the four rows
template <int DHP> __device__ __forceinline__ unsigned pa_col_place() {
    typedef PaTile<DHP> TL;
    const int lane = threadIdx.x & 63, li = lane & 15, row = 4 * (lane >> 5) + (li >> 2), col = 16 * ((lane >> 4) & 1) + 4 * (li & 3);
    return row * TL::RB + (((col >> 3) ^ TL::swz(row)) << 4) + (col & 7) * 2;
}
template <typename V8, int DHP> __device__ __forceinline__ V8 pa_col_frag(const char* lds, unsigned place, int r0, int mt) {
    typedef PaTile<DHP> TL;
    const char* const p = lds + r0 * TL::RB;
    const unsigned at = place ^ (mt << 6);                                 // (eight rows on, bit 1 of the xor is the other one)
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(p + at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(p + 8 * TL::RB + (at ^ 32)));
    const s16x8 r = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(V8, r);
}
// ds as a 32-bit number: in fp16 the compiler would take the 16-bit part straight from the product of its factors (one rounding, v_fma_mix) and the rest
// from the product in 32 bits (two), which differ by a whole step once in some thousand pairs
template <typename T> __device__ __forceinline__ void pa_settle(float (&ds)[16]) {
    if constexpr (std::is_same<T, f16>::value) {
#pragma unroll
        for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(ds[i]));
    }
}
// Operands in fp16 lie within its normal numbers, 2^-14 to 65504, or lose bits; probabilities and ds of long rows do not: about 1 / keys, and that times
// the output gradient.  So p carries a factor of 2^12 in the pass over keys (it is at most 1), and ds a power of two per owned row, i.e. per lane:
// `up` brings the row's largest ds so far between 2^8 and 2^15, falls when a larger one comes, the row's accumulators with it, and is taken out
// of the result.  Powers of two round nothing.  bf16 has the exponents of 32 bits and takes neither.  Without it dq's error is 6.9 times what the
// roundings explain with output gradients of 1e-3, 4096 keys and heads of 64 (ds down to 2^-24 steps); it costs the fp16 backward pass 4 to 11 % (batch of
// 2048 ... 1 causal tokens, 16 heads of 128 over 4: 330 -> 343 us), 13 % with heads of 32.
template <typename T> struct PaRange { static constexpr float P_LOG = 0.f, P_OFF = 1.f, UP = 1.f; };
template <> struct PaRange<f16> { static constexpr float P_LOG = 12.f, P_OFF = 0x1p-12f, UP = 0x1p60f; };
template <typename T, int MT> __device__ __forceinline__ void pa_raise(float (&ds)[16], float& up, f32x16 (&acc)[MT]) {
    if constexpr (std::is_same<T, f16>::value) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(ds[i]));
        top = pa_half_max(top);
        if (__any(top * up > 0x1p15f)) {
            // 2^8 / the power of two in top (its exponent is at least -45 here, at most 128 for infinity)
            const unsigned to = top * up > 0x1p15f ? (262u - (__float_as_uint(top) >> 23)) << 23 : __float_as_uint(up);
            const float by = __builtin_amdgcn_ldexpf(1.f, (int)(to >> 23) - (int)(__float_as_uint(up) >> 23));
            up = __uint_as_float(to);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[mt][i] *= by;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[i] *= up;
    }
}
template <int DHP> __device__ __forceinline__ void pa_opaque(unsigned& place) {
    if constexpr (DHP == 128) asm volatile("" : "+v"(place));
}

// A wave's own rows (up to 32, from row `row`, one a lane) through a buffer that ends with the last of them: what is out of range reads as
// zeros and is not written, so that neither rows that do not exist nor pieces past the head's width need a branch.
struct PaOwn {
    __amdgpu_buffer_rsrc_t buffer;
    unsigned at;                                                           // of the lane's row, in bytes
    int dh;
    bool valid;
};
__device__ __forceinline__ PaOwn pa_rows(const PaView& x, long long row, int rows, int head, int dh) {
    const unsigned bytes = rows > 0 ? (unsigned)((rows - 1) * x.row + dh) * 2u : 0u;
    const int col = threadIdx.x & 31;
    return {__builtin_amdgcn_make_buffer_rsrc((char*)x.p + (row * x.row + head * x.head) * 2, 0, bytes, 0x00020000), (unsigned)(col * x.row) * 2u, dh, col < rows};
}
// as operands: elements kc*16 + h*8 ... + 7
template <typename V8, int DHP> __device__ __forceinline__ void pa_own(V8 (&f)[DHP / 16], const PaOwn& x) {
#pragma unroll
    for (int kc = 0; kc < DHP / 16; ++kc) {
        const int d = kc * 16 + (int)((threadIdx.x >> 5) & 1) * 8;
        f[kc] = __builtin_bit_cast(V8, __builtin_amdgcn_raw_buffer_load_b128(x.buffer, x.valid && d < x.dh ? x.at + d * 2u : 0xfffffff0u, 0, 0));
    }
}
// a transposed result (rows = head dimensions, column = the lane's row)
template <typename T, int DHP, typename F> __device__ __forceinline__ void pa_put(const f32x16 (&acc)[DHP / 32], const PaOwn& x, F&& f) {
    typedef typename PaTypes<T>::v4 v4;
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int mt = 0; mt < DHP / 32; ++mt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = mt * 32 + g * 8 + (int)((threadIdx.x >> 5) & 1) * 4;
            v4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = (T)f(acc[mt][g * 4 + j]);
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, w), x.buffer, x.valid && d < x.dh ? x.at + d * 2u : 0xfffffff0u, 0, 0);
        }
}

template <typename T> __device__ __forceinline__ typename PaTypes<T>::v8 pa_pack(const float* s) {
    typename PaTypes<T>::v8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)s[j];
    return r;
}

// what rounding to T leaves of it, rounded: a second product with this takes the probabilities to about 2^-16 (bf16), 2^-22 (fp16)
template <typename T> __device__ __forceinline__ typename PaTypes<T>::v8 pa_rest(const float* s) {
    typename PaTypes<T>::v8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)(s[j] - (float)(T)s[j]);
    return r;
}

// ---- relative position bias ----------------------------------------------------------------------------------------------------
// LDS: the bias of every distance key - query in -far ... far for one head, in units of log2 like the scores.  Finite ones are limited to
// PA_MAX_BIAS: a row all of whose keys have the same large bias keeps its scores and its normaliser in 32 bits (with a bias of -1e9 both
// would be lost, and the backward pass could not rebuild the probabilities).  -inf stays: a distance that is not seen.
#define PA_MAX_BIAS 8192.f
__device__ __forceinline__ void pa_bias_fill(const PaArgs& a, int head, float* s_bias) {
    for (int i = threadIdx.x; i < 2 * a.far + 1; i += blockDim.x) {
        int b = a.bucket_of[i];
        b = b < 0 ? 0 : b >= a.buckets ? a.buckets - 1 : b;
        const float t = a.table[(long long)b * a.H + head], x = t * 1.4426950408889634f;
        s_bias[i] = fabsf(t) < INFINITY ? fminf(fmaxf(x, -PA_MAX_BIAS), PA_MAX_BIAS) : x;
    }
}
__device__ __forceinline__ int pa_clamp(int d, int far) { return d < -far ? -far : d > far ? far : d; }

// ================================================================================================================================
// forward
// ================================================================================================================================
// TWO: with a bias whose gradient will be wanted, from p in two parts
template <typename T, int DHP, bool BIAS, bool TWO>
__global__ __launch_bounds__(256, 2) void pa_fwd_kernel(const PaArgs a) {
    typedef typename PaTypes<T>::v8 v8;
    typedef PaTile<DHP> TL;
    constexpr int KC = DHP / 16, MT = DHP / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // k, v tiles, two buffers of both; then the bias
    float* const s_bias = (float*)(smem + 4 * TL::BYTES);
    // heads that share k, v differ by Hk in their index: with workgroups dealt to the eight XCDs in turn, they meet in one L2
    const int hk = blockIdx.x % a.Hk, g = blockIdx.x / a.Hk % (a.H / a.Hk), head = hk * (a.H / a.Hk) + g;
    PaSeq sq;
    if (!pa_find<false>(a.ends_q, a.Tq, a.ends_k, a.Tk, a.B, a.zero_rest, a.causal, (int)(blockIdx.x / a.H), a.slots, sq)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    const int w0 = sq.row0 + wave * 32, qi = w0 + col;                     // the wave's first row, the lane's row
    const bool qv = qi < sq.n;
    const int off = a.causal ? sq.n2 - sq.n : 0;                           // a causal row's last key is row + off
    if (BIAS) pa_bias_fill(a, head, s_bias);

    const int w_rows = sq.n - w0 < 32 ? sq.n - w0 : 32;                    // <= 0: the wave has no rows
    v8 bq[KC];
    pa_own<v8, DHP>(bq, pa_rows(a.q, sq.begin + w0, w_rows, head, a.dh));
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
    const unsigned ko = pa_piece<DHP>(a.k.row, a.dh), vo = pa_piece<DHP>(a.v.row, a.dh);
    auto fetch = [&](int t) {
        const unsigned to = pa_lds(smem) + (t & 1) * 2 * TL::BYTES;
        pa_load<DHP, PA_TILE>(to, kb, a.k.row, t * PA_TILE, sq.n2, a.dh, ko);
        pa_load<DHP, PA_TILE>(to + TL::BYTES, vb, a.v.row, t * PA_TILE, sq.n2, a.dh, vo);
    };
    if (tiles > 0) fetch(0);
    unsigned rp = pa_row_place<DHP>(col, h), cp = pa_col_place<DHP>();
    const int seen = a.causal ? w0 + w_rows - 1 + off : sq.n2 - 1;         // the last key that a row of the wave sees
    const int mine = w_rows > 0 && seen >= 0 ? (seen / PA_TILE + 1 < tiles ? seen / PA_TILE + 1 : tiles) : 0;
    auto arrive = [&](int t) {
        pa_arrived();
        __syncthreads();                                                   // this tile is there, and the one before it has been read
        if (t + 1 < tiles) fetch(t + 1);
    };
    // (tiles that the wave has no part in, all behind its own, have a loop of their own: as a branch in this one they made the compiler move the
    // accumulators to other registers and back for every tile, 64 instructions: 4 % of the time of 16 K causal tokens)
    for (int t = 0; t < mine; ++t) {
        if (BIAS) {
            pa_opaque<DHP>(rp);
            pa_opaque<DHP>(cp);
        }
        const char* const lk = smem + (t & 1) * 2 * TL::BYTES;
        const char* const lv = lk + TL::BYTES;
        const int k0 = t * PA_TILE;
        arrive(t);
        f32x16 sc[2] = {pa_zero(), pa_zero()};
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            sc[0] = pa_mfma(pa_row_frag<v8, DHP>(lk, rp, kc), bq[kc], sc[0]);
            sc[1] = pa_mfma(pa_row_frag<v8, DHP>(lk + 32 * TL::RB, rp, kc), bq[kc], sc[1]);
        }
        pa_order<2 * KC, 1, 4>();
        __builtin_amdgcn_s_setprio(0);
        float s[32];
        const int dist0 = k0 + h * 4 - (qi + off);                     // distance of the lane's first score
        if (BIAS) {
            const int lo = k0 - (w0 + 31 + off), hi = k0 + PA_TILE - 1 - (w0 + off);       // distances in the wave's tile
            if (hi <= -a.far || lo >= a.far) {
                const float b = s_bias[hi <= -a.far ? 0 : 2 * a.far];
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = sc[i >> 4][i & 15] * a.scale2 + b;
            } else if (lo > -a.far && hi < a.far) {                    // no distance is clamped: one address, constant offsets
                const float* const b = s_bias + dist0 + a.far;
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = sc[i >> 4][i & 15] * a.scale2 + b[(i >> 2) * 8 + (i & 3)];
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    s[i] = sc[i >> 4][i & 15] * a.scale2 + s_bias[pa_clamp(dist0 + (i >> 2) * 8 + (i & 3), a.far) + a.far];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i] = sc[i >> 4][i & 15];    // (scaled where the maximum is subtracted, in one instruction)
        }
        if (k0 + PA_TILE > sq.n2 || (a.causal && k0 + PA_TILE - 1 > w0 + off)) {
            // key index - k0 of score i is (i >> 2) * 8 + h * 4 + (i & 3): beyond `last` it is not seen
            const int last = (a.causal && qi + off < sq.n2 - 1 ? qi + off : sq.n2 - 1) - k0 - h * 4;
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i] = (i >> 2) * 8 + (i & 3) <= last ? s[i] : -INFINITY;
        }
        const float unit = BIAS ? 1.f : a.scale2;                      // (positive: the maximum may be taken before)
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 32; ++i) mx = fmaxf(mx, s[i]);
        mx = pa_half_max(mx) * unit;
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
            s[i] = __builtin_amdgcn_exp2f(s[i] * unit - ref);
            sum += s[i];
        }
        l += sum;                                                      // (this half-wave's keys; joined at the end)
        // p is rounded to the type of v for the product (relative 2^-8 of each term in bf16, of either sign); the sum above is not.
        // Where the output feeds the bias's gradient, whose terms cancel, what that rounding leaves is multiplied as well.
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const v8 p = pa_pack<T>(s + 8 * c);
            v8 rest;
            if constexpr (TWO) rest = pa_rest<T>(s + 8 * c);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const v8 f = pa_col_frag<v8, DHP>(lv, cp, 16 * c, mt);
                acc[mt] = pa_mfma(f, p, acc[mt]);
                if constexpr (TWO) acc[mt] = pa_mfma(f, rest, acc[mt]);
            }
        }
        if (!TWO) pa_order<4 * MT, 2, 3>();
        __builtin_amdgcn_s_setprio(0);
    }
    for (int t = mine; t < tiles; ++t) arrive(t);
    l = pa_half_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    pa_put<T, DHP>(acc, pa_rows(a.o, sq.begin + w0, w_rows, head, a.dh), [&](float x) { return x * inv; });
    if (!qv) return;
    const long long row = sq.begin + qi;
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
// The gradient of the bias is a sum of ds over equal distances first and over the distances of a bucket last.  A tile wholly at
// distances beyond -far or far adds to two registers.  Of other tiles, 16 keys at a time go to LDS and come back by diagonals, a lane to
// each, whose sums a wave adds to an array of its own (1.5 us of a workgroup's time for a tile's 16 registers as LDS atomics, which is
// what fp32 ones cost; this way 0.1).  Every sum has a fixed order and is taken from the 32-bit ds.
//   D.  Where the workgroup's rows see at most two tiles of keys, D = sum_j p_ij (do_i . v_j) comes from a sweep over those: their
// ds are few and of D's own size, and the rounding of o would be the largest error of dq (3e-3 of it instead of 2.4e-3 in bf16).  Longer
// rows take do . o.  The sum of a row's ds, zero for the exact D, then says by how much that D was off: dk and the bias's gradient at
// far distances (most of a long row) are corrected by it, and o comes in 32 bits with p in two parts there (1e-6 of the bias's
// gradient instead of 5e-4).
template <typename T, int DHP, bool BIAS>
__global__ __launch_bounds__(256, 2) void pa_bwd_dq_kernel(const PaArgs a) {
    typedef typename PaTypes<T>::v8 v8;
    typedef PaTile<DHP> TL;
    constexpr int KC = DHP / 16, MT = DHP / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // k, v tiles, two buffers of both; then the bias and its sums
    const int width = 2 * a.far + 1;
    float* const s_bias = (float*)(smem + 4 * TL::BYTES);
    float* const s_sum = s_bias + width;                                   // [4][width]
    const int hk = blockIdx.x % a.Hk, g = blockIdx.x / a.Hk % (a.H / a.Hk), head = hk * (a.H / a.Hk) + g;
    const int rank = (int)(blockIdx.x / a.H);
    const bool want_table = BIAS && a.dtable_part;
    float* const part = want_table ? a.dtable_part + ((long long)rank * a.H + head) * a.buckets : nullptr;
    PaSeq sq;
    if (!pa_find<false>(a.ends_q, a.Tq, a.ends_k, a.Tk, a.B, a.zero_rest, a.causal, rank, a.slots, sq)) {
        if (want_table)
            for (int i = threadIdx.x; i < a.buckets; i += 256) part[i] = 0.f;
        return;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    const int w0 = sq.row0 + wave * 32, qi = w0 + col;
    const bool qv = qi < sq.n;
    const int off = a.causal ? sq.n2 - sq.n : 0;
    const long long row = sq.begin + (qv ? qi : 0);
    if (BIAS) {
        pa_bias_fill(a, head, s_bias);
        if (want_table)
            for (int i = threadIdx.x; i < 4 * width; i += 256) s_sum[i] = 0.f;
    }
    float* const my_sum = s_sum + wave * width, *const s_tile = s_sum + 4 * width + wave * (32 * 17);   // the tile: [query][key], 17 apart
    // bit kk: the lane's diagonal has an element at key kk, 0 <= kk + 31 - lane <= 31
    const int on_tile = lane <= 31 ? (2 << lane) - 1 : lane < 63 ? -1 << (lane - 31) : 0;
    float before = 0.f, after = 0.f, pbefore = 0.f, pafter = 0.f;          // ds and p at distances <= -far, >= far
    float all = 0.f;                                                       // every ds of the row
    float up = PaRange<T>::UP;

    const int w_rows = sq.n - w0 < 32 ? sq.n - w0 : 32;
    v8 bq[KC], bdo[KC];
    pa_own<v8, DHP>(bq, pa_rows(a.q, sq.begin + w0, w_rows, head, a.dh));
    pa_own<v8, DHP>(bdo, pa_rows(a.dout, sq.begin + w0, w_rows, head, a.dh));
    const int rows = sq.n - sq.row0 < PA_ROWS ? sq.n - sq.row0 : PA_ROWS;
    int keys = a.causal ? sq.row0 + rows + off : sq.n2;
    keys = keys < 0 ? 0 : keys < sq.n2 ? keys : sq.n2;
    const int tiles = (keys + PA_TILE - 1) / PA_TILE;
    const bool sweep = tiles <= 2;
    // ds in two parts where its rounding shows: few keys, whose terms do not average out, and narrow heads, whose weighted mean of the keys
    // is not small against the keys and cancels (the sum of a row's ds is zero).  dq's error, in multiples of one rounding of the result: 1.4 to 2.6
    // with one part and few keys, 1.6 with heads of 8; 1.0 with two.  (The branch costs long rows of wide heads 2 %.)
    const bool two = sweep || DHP == 32;
    // (-inf: no key seen, as where a bias of -inf hides all of them.  As +inf, every probability comes out as zero; -inf - -inf would be NaN)
    float lse = qv ? a.lse[(long long)head * a.Tq + row] : 0.f;
    if (lse == -INFINITY) lse = INFINITY;
    float dsum = 0.f;
    if (sweep) {
    } else if (a.o32) {
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
        pa_own<v8, DHP>(of, pa_rows(a.o, sq.begin + w0, w_rows, head, a.dh));
#pragma unroll
        for (int kc = 0; kc < KC; ++kc)
#pragma unroll
            for (int j = 0; j < 8; ++j) dsum += (float)bdo[kc][j] * (float)of[kc][j];
    }
    dsum = pa_half_sum(dsum);
    f32x16 acc[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt] = pa_zero();

    const char* const kb = (const char*)a.k.p + (sq.begin2 * a.k.row + hk * a.k.head) * 2;
    const char* const vb = (const char*)a.v.p + (sq.begin2 * a.v.row + hk * a.v.head) * 2;
    const unsigned ko = pa_piece<DHP>(a.k.row, a.dh), vo = pa_piece<DHP>(a.v.row, a.dh);
    auto fetch = [&](int t) {
        const unsigned to = pa_lds(smem) + (t & 1) * 2 * TL::BYTES;
        pa_load<DHP, PA_TILE>(to, kb, a.k.row, t * PA_TILE, sq.n2, a.dh, ko);
        pa_load<DHP, PA_TILE>(to + TL::BYTES, vb, a.v.row, t * PA_TILE, sq.n2, a.dh, vo);
    };
    unsigned rp = pa_row_place<DHP>(col, h), cp = pa_col_place<DHP>();
    // probabilities (zero where the key is not seen) and from + do . v of 32 keys
    auto scores = [&](const char* lk, const char* lv, int sub, int k0, float (&p)[16], f32x16& dp, const f32x16& from) {
        f32x16 sc = pa_zero();
        dp = from;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            sc = pa_mfma(pa_row_frag<v8, DHP>(lk + sub * 32 * TL::RB, rp, kc), bq[kc], sc);
            dp = pa_mfma(pa_row_frag<v8, DHP>(lv + sub * 32 * TL::RB, rp, kc), bdo[kc], dp);
        }
        pa_order<2 * KC, 1, 4>();
        __builtin_amdgcn_s_setprio(0);
        const int dist0 = k0 + h * 4 - (qi + off), lo = k0 - (w0 + 31 + off), hi = k0 + 31 - (w0 + off);
        if (!BIAS || hi <= -a.far || lo >= a.far) {
            const float b = BIAS ? s_bias[hi <= -a.far ? 0 : 2 * a.far] - lse : -lse;
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(sc[i] * a.scale2 + b);
        } else if (lo > -a.far && hi < a.far) {                            // no distance is clamped: one address, constant offsets
            const float* const b = s_bias + dist0 + a.far;
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(sc[i] * a.scale2 + (b[(i >> 2) * 8 + (i & 3)] - lse));
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                p[i] = __builtin_amdgcn_exp2f(sc[i] * a.scale2 + (s_bias[pa_clamp(dist0 + (i >> 2) * 8 + (i & 3), a.far) + a.far] - lse));
        }
        if (k0 + 32 > sq.n2 || w_rows < 32 || (a.causal && k0 + 31 > w0 + off)) {
            int last = (a.causal && qi + off < sq.n2 - 1 ? qi + off : sq.n2 - 1) - k0 - h * 4;
            if (!qv) last = -1;
#pragma unroll
            for (int i = 0; i < 16; ++i) {                                 // (do . v of a key that is not seen may be anything)
                p[i] = (i >> 2) * 8 + (i & 3) <= last ? p[i] : 0.f;
                dp[i] = (i >> 2) * 8 + (i & 3) <= last ? dp[i] : 0.f;
            }
        }
    };
    auto sees = [&](int k0) { return w_rows > 0 && k0 < sq.n2 && (!a.causal || k0 <= w0 + w_rows - 1 + off); };

    if (tiles > 0) fetch(0);
    if (sweep) {
        if (tiles == 2) fetch(1);
        pa_arrived();
        __syncthreads();
        for (int u = 0; u < 2 * tiles; ++u) {
            const char* const lk = smem + (u >> 1) * 2 * TL::BYTES;
            if (sees(u * 32)) {
                float p[16];
                f32x16 dp;
                scores(lk, lk + TL::BYTES, u & 1, u * 32, p, dp, pa_zero());
#pragma unroll
                for (int i = 0; i < 16; ++i) dsum += p[i] * dp[i];
            }
        }
        dsum = pa_half_sum(dsum);
    }
    f32x16 minus_d;                                                        // do . v - D: the products begin with -D, sixteen registers that never change
#pragma unroll
    for (int i = 0; i < 16; ++i) minus_d[i] = -dsum;
    for (int t = 0; t < tiles; ++t) {
        const char* const lk = smem + (t & 1) * 2 * TL::BYTES;
        const char* const lv = lk + TL::BYTES;
        pa_opaque<DHP>(rp);
        pa_opaque<DHP>(cp);
        if (!sweep) {
            pa_arrived();
            __syncthreads();                                               // this tile is there, and the one before it has been read
            if (t + 1 < tiles) fetch(t + 1);
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int k0 = t * PA_TILE + sub * 32;
            if (sees(k0)) {
                float p[16], ds[16], sum = 0.f;
                f32x16 dp;
                scores(lk, lv, sub, k0, p, dp, minus_d);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    ds[i] = p[i] * dp[i];
                    sum += ds[i];
                }
                pa_settle<T>(ds);
                all += sum;
                if (want_table) {
                    const int lo = k0 - (w0 + 31 + off), hi = k0 + 31 - (w0 + off);
                    if (hi <= -a.far || lo >= a.far) {
                        float ps = 0.f;
#pragma unroll
                        for (int i = 0; i < 16; ++i) ps += p[i];
                        if (lo >= a.far) { after += sum; pafter += ps; }
                        else { before += sum; pbefore += ps; }
                    } else {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            pa_wave_order();
#pragma unroll
                            for (int i = 0; i < 8; ++i) s_tile[col * 17 + (i >> 2) * 8 + h * 4 + (i & 3)] = ds[half * 8 + i];
                            pa_wave_order();
                            // lane's diagonal: key - query = lane - 31; what a lane reads off the tile's ends is dropped, by bits (as
                            // conditions they became sixteen branches around sixteen reads that waited for each other)
                            const float* const at = s_tile + (31 - lane) * 17;
                            float e[16], x = 0.f;
#pragma unroll
                            for (int kk = 0; kk < 16; ++kk) e[kk] = at[kk * 18];
#pragma unroll
                            for (int kk = 0; kk < 16; ++kk) x += __int_as_float(__float_as_int(e[kk]) & __builtin_amdgcn_sbfe(on_tile, kk, 1));
                            const int d = k0 + half * 16 - (w0 + off) + lane - 31;
                            before += d <= -a.far ? x : 0.f;
                            after += d >= a.far ? x : 0.f;
                            if (d > -a.far && d < a.far && lane < 47) my_sum[d + a.far] += x;
                        }
                    }
                }
                // ds is rounded to the type of k for the product (see p in the forward pass)
                pa_raise<T, MT>(ds, up, acc);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const v8 r = pa_pack<T>(ds + 8 * c);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) acc[mt] = pa_mfma(pa_col_frag<v8, DHP>(lk, cp, sub * 32 + 16 * c, mt), r, acc[mt]);
                }
                pa_order<2 * MT, 2, 3>();
                __builtin_amdgcn_s_setprio(0);
                if (two) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const v8 r = pa_rest<T>(ds + 8 * c);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) acc[mt] = pa_mfma(pa_col_frag<v8, DHP>(lk, cp, sub * 32 + 16 * c, mt), r, acc[mt]);
                    }
                }
            }
        }
    }
    all = pa_half_sum(all);
    if (qv && h == 0) a.dsum[(long long)head * a.Tq + row] = dsum + all;
    const float out = a.scale / up;
    pa_put<T, DHP>(acc, pa_rows(a.dq, sq.begin + w0, w_rows, head, a.dh), [&](float x) { return x * out; });
    if (!want_table) return;
    before = wave_sum(before - all * pbefore);
    after = wave_sum(after - all * pafter);
    __syncthreads();
    if (lane == 0) { s_bias[wave * 2] = before; s_bias[wave * 2 + 1] = after; }       // (the bias itself is no longer needed; width >= 9)
    __syncthreads();
    for (int i = threadIdx.x; i < width; i += 256) {
        float x = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) x += s_sum[k * width + i];
        if (i == 0) x += (s_bias[0] + s_bias[2]) + (s_bias[4] + s_bias[6]);
        if (i == 2 * a.far) x += (s_bias[1] + s_bias[3]) + (s_bias[5] + s_bias[7]);
        int k = a.bucket_of[i];
        k = k < 0 ? 0 : k >= a.buckets ? a.buckets - 1 : k;
        s_sum[i] = x;                                  // (only this thread reads or writes column i of the four)
        s_sum[width + i] = __int_as_float(k);
    }
    __syncthreads();
    // eight lanes take a bucket, each every eighth distance
    for (int b0 = 0; b0 < a.buckets; b0 += 32) {
        const int b = b0 + (threadIdx.x >> 3);
        float x = 0.f;
#pragma unroll 4
        for (int i = threadIdx.x & 7; i < width; i += 8) x += __float_as_int(s_sum[width + i]) == b ? s_sum[i] : 0.f;
        for (int o = 1; o < 8; o <<= 1) x += __shfl_xor(x, o, 64);
        if ((threadIdx.x & 7) == 0 && b < a.buckets) part[b] = x;
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
// Heads of 128: the accumulators and k take 160 registers, so that v is read from LDS and tiles are 32 queries, which leaves room for two
// workgroups on a CU, each waiting at barriers of its own (one workgroup with v in registers and tiles of 64 queries took twice as long for the batch of
// 2048 ... 1 causal tokens, 16 heads over 4, which takes 199 to 220 us now).
// The steps (heads of the group x tiles of queries) may be split over several workgroups, whose 32-bit sums a last launch adds
// up: few keys with long sequences and shared heads would leave most of the card idle otherwise.
template <typename T, int DHP, bool BIAS>
__global__ __launch_bounds__(256, 2) void pa_bwd_dkv_kernel(const PaArgs a) {
    typedef typename PaTypes<T>::v8 v8;
    constexpr int KC = DHP / 16, MT = DHP / 32;
    constexpr int ROWS = DHP == 128 ? 32 : PA_TILE;
    constexpr bool VLDS = DHP == 128;
    typedef PaTile<DHP, ROWS> TL;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // q, do tiles, two buffers of both; lse and D of their rows; the bias
    float* const s_row = (float*)(smem + 4 * TL::BYTES);                   // [2][2][ROWS]
    float* const s_bias = s_row + 4 * ROWS;
    const int hk = blockIdx.x % a.Hk, group = a.H / a.Hk;
    const int split = __builtin_amdgcn_readfirstlane((int)(blockIdx.x / a.Hk % a.splits));
    PaSeq sq;                                                              // begin, n: keys; begin2, n2: queries
    if (!pa_find<true>(a.ends_k, a.Tk, a.ends_q, a.Tq, a.B, a.zero_rest, a.causal, (int)(blockIdx.x / (a.Hk * a.splits)), a.slots, sq)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    const int w0 = sq.row0 + wave * 32, ki = w0 + col;
    const bool kv = ki < sq.n;
    const int off = a.causal ? sq.n - sq.n2 : 0;
    const int w_rows = sq.n - w0 < 32 ? sq.n - w0 : 32;
    char* const s_v = smem + 4 * TL::BYTES + 16 * ROWS + (BIAS ? ((2 * a.far + 1) * 4 + 15) / 16 * 16 : 0);
    v8 bk[KC], bv[KC];
    pa_own<v8, DHP>(bk, pa_rows(a.k, sq.begin + w0, w_rows, hk, a.dh));
    pa_own<v8, DHP>(bv, pa_rows(a.v, sq.begin + w0, w_rows, hk, a.dh));
    if (VLDS) {
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) *(v8*)(s_v + wave * 32 * TL::RB + (pa_row_place<DHP>(col, h) ^ (kc << 5))) = bv[kc];
    }
    f32x16 dk[MT], dv[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) { dk[mt] = pa_zero(); dv[mt] = pa_zero(); }
    int first = a.causal ? sq.row0 - off : 0;                              // the first query that sees any key of the workgroup
    first = first < 0 ? 0 : first / ROWS * ROWS;
    const int tiles = sq.n2 > first ? (sq.n2 - first + ROWS - 1) / ROWS : 0;
    const bool two = sq.n2 <= 2 * PA_TILE || DHP == 32;                    // p and ds in two parts: few queries, narrow heads (see the pass over queries)
    const int steps = tiles * group, share = __builtin_amdgcn_readfirstlane((steps + a.splits - 1) / a.splits);
    const int begin = split * share < steps ? split * share : steps, end = begin + share < steps ? begin + share : steps;
    const unsigned qo = pa_piece<DHP>(a.q.row, a.dh), po = pa_piece<DHP>(a.dout.row, a.dh);
    float up = PaRange<T>::UP;
    float rst = 0.f;                                                       // the first ROWS threads: lse of a query, the next: its -D
    // the step that is loaded next: head hd, tile td
    int hd = tiles > 0 ? __builtin_amdgcn_readfirstlane(begin / tiles) : 0, td = begin - hd * tiles;
    auto fetch = [&](int buf) {
        const int head = hk * group + hd, q0 = first + td * ROWS;
        const unsigned to = pa_lds(smem) + buf * 2 * TL::BYTES;
        pa_load<DHP, ROWS>(to, (const char*)a.q.p + (sq.begin2 * a.q.row + head * a.q.head) * 2, a.q.row, q0, sq.n2, a.dh, qo);
        pa_load<DHP, ROWS>(to + TL::BYTES, (const char*)a.dout.p + (sq.begin2 * a.dout.row + head * a.dout.head) * 2, a.dout.row, q0, sq.n2, a.dh, po);
        if (threadIdx.x < 2 * ROWS) {
            const int q = q0 + (threadIdx.x & (ROWS - 1));
            const long long at = (long long)head * a.Tq + sq.begin2 + q;
            if (threadIdx.x < ROWS) {
                rst = q < sq.n2 ? a.lse[at] - PaRange<T>::P_LOG : INFINITY;
                if (rst == -INFINITY) rst = INFINITY;                      // no key seen, or no query: every probability comes out as zero
            } else
                rst = q < sq.n2 ? -a.dsum[at] : 0.f;
        }
        if (++td == tiles) { td = 0; ++hd; }
    };
    auto keep = [&](int buf) {
        if (threadIdx.x < 2 * ROWS) s_row[buf * 2 * ROWS + threadIdx.x] = rst;
    };
    int q_head = hd, q_tile = td;                                          // the step that is computed next
    if (begin < end) {
        fetch(begin & 1);
        keep(begin & 1);
    }
    unsigned rp = pa_row_place<DHP>(col, h), cp = pa_col_place<DHP>(), vp = wave * 32 * TL::RB + rp;
    for (int step = begin; step < end; ++step) {
        pa_opaque<DHP>(rp);
        pa_opaque<DHP>(cp);
        pa_opaque<DHP>(vp);
        if (BIAS && (step == begin || q_tile == 0)) {
            __syncthreads();
            pa_bias_fill(a, hk * group + q_head, s_bias);
        }
        pa_arrived();
        __syncthreads();                                                   // this tile is there, and the one before it has been read
        const char* const lq = smem + (step & 1) * 2 * TL::BYTES;
        const char* const lp = lq + TL::BYTES;
        if (step + 1 < end) fetch((step + 1) & 1);
#pragma unroll
        for (int sub = 0; sub < ROWS / 32; ++sub) {
        const float* const lr = s_row + (step & 1) * 2 * ROWS + sub * 32 + h * 4;
        const int q0 = first + q_tile * ROWS + sub * 32;
        if (w_rows > 0 && q0 < sq.n2 && (!a.causal || q0 + 31 + off >= w0)) {
            f32x16 sc = pa_zero(), dp;                                     // dp: do . v - D, begun with -D
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 dd = *(const f32x4*)(lr + ROWS + g * 8);
#pragma unroll
                for (int j = 0; j < 4; ++j) dp[g * 4 + j] = dd[j];
            }
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) sc = pa_mfma(pa_row_frag<v8, DHP>(lq + sub * 32 * TL::RB, rp, kc), bk[kc], sc);
#pragma unroll
            for (int kc = 0; kc < KC; ++kc)
                dp = pa_mfma(pa_row_frag<v8, DHP>(lp + sub * 32 * TL::RB, rp, kc), VLDS ? pa_row_frag<v8, DHP>(s_v, vp, kc) : bv[kc], dp);
            pa_order<KC, 1, 3>();
            pa_order<KC, VLDS ? 2 : 1, 2>();
            __builtin_amdgcn_s_setprio(0);
            // (here, so that a branch ends the region in which the compiler may hold these products back and keep all their operands instead)
            if (a.causal && w0 + w_rows - 1 > q0 + off) {
                const int firstq = ki - off - q0 - h * 4;                  // query index of a row that sees this key
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sc[i] = (i >> 2) * 8 + (i & 3) >= firstq ? sc[i] : -INFINITY;
                    dp[i] = (i >> 2) * 8 + (i & 3) >= firstq ? dp[i] : 0.f;
                }
            }
            float p[16];
            const int dist0 = ki - (q0 + h * 4 + off), lo = w0 - (q0 + 31 + off), hi = w0 + 31 - (q0 + off);   // distance of the lane's first score; later rows are nearer
            if (!BIAS) {
            } else if (hi <= -a.far || lo >= a.far) {
                const float b = s_bias[hi <= -a.far ? 0 : 2 * a.far];
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = sc[i] * a.scale2 + b;
            } else if (lo > -a.far && hi < a.far) {
                const float* const b = s_bias + dist0 + a.far;
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = sc[i] * a.scale2 + b[-((i >> 2) * 8 + (i & 3))];
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = sc[i] * a.scale2 + s_bias[pa_clamp(dist0 - ((i >> 2) * 8 + (i & 3)), a.far) + a.far];
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 ls = *(const f32x4*)(lr + g * 8);
#pragma unroll
                for (int j = 0; j < 4; ++j) p[g * 4 + j] = __builtin_amdgcn_exp2f(BIAS ? p[g * 4 + j] - ls[j] : sc[g * 4 + j] * a.scale2 - ls[j]);
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const v8 r = pa_pack<T>(p + 8 * c);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) dv[mt] = pa_mfma(pa_col_frag<v8, DHP>(lp, cp, sub * 32 + 16 * c, mt), r, dv[mt]);
            }
            pa_order<2 * MT, 2, 3>();
            if (two) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const v8 r = pa_rest<T>(p + 8 * c);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) dv[mt] = pa_mfma(pa_col_frag<v8, DHP>(lp, cp, sub * 32 + 16 * c, mt), r, dv[mt]);
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] *= dp[i];
            pa_settle<T>(p);
            pa_raise<T, MT>(p, up, dk);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const v8 r = pa_pack<T>(p + 8 * c);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) dk[mt] = pa_mfma(pa_col_frag<v8, DHP>(lq, cp, sub * 32 + 16 * c, mt), r, dk[mt]);
            }
            pa_order<2 * MT, 2, 3>();
            __builtin_amdgcn_s_setprio(0);
            if (two) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const v8 r = pa_rest<T>(p + 8 * c);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) dk[mt] = pa_mfma(pa_col_frag<v8, DHP>(lq, cp, sub * 32 + 16 * c, mt), r, dk[mt]);
                }
            }
        }
        }
        if (++q_tile == tiles) { q_tile = 0; ++q_head; }
        if (step + 1 < end) keep((step + 1) & 1);
    }
    const float k_out = PaRange<T>::P_OFF / up;
    if (a.dkv_part) {
        if (!kv) return;
        const long long row = sq.begin + ki;
        float* const p = a.dkv_part + (((long long)split * a.Tk + row) * a.Hk + hk) * a.dh, *const p2 = p + (long long)a.splits * a.Tk * a.Hk * a.dh;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = mt * 32 + g * 8 + h * 4;
                if (d < a.dh) {
                    *(f32x4*)(p + d) = f32x4{dk[mt][g * 4], dk[mt][g * 4 + 1], dk[mt][g * 4 + 2], dk[mt][g * 4 + 3]} * k_out;
                    *(f32x4*)(p2 + d) = f32x4{dv[mt][g * 4], dv[mt][g * 4 + 1], dv[mt][g * 4 + 2], dv[mt][g * 4 + 3]} * PaRange<T>::P_OFF;
                }
            }
        return;
    }
    pa_put<T, DHP>(dk, pa_rows(a.dk, sq.begin + w0, w_rows, hk, a.dh), [&](float x) { return x * (a.scale * k_out); });
    pa_put<T, DHP>(dv, pa_rows(a.dv, sq.begin + w0, w_rows, hk, a.dh), [&](float x) { return x * PaRange<T>::P_OFF; });
}

// dk, dv = the sums over the splits, in order: a thread takes four elements of a row of both
template <typename T> __global__ __launch_bounds__(256) void pa_dkv_join_kernel(const PaArgs a) {
    typedef typename PaTypes<T>::v4 v4;
    const int per = a.Hk * (a.dh / 4);
    const long long idx = blockIdx.x * 256ll + threadIdx.x, total = (long long)a.Tk * per;
    if (idx >= total) return;
    const int row = (int)(idx / per), c = (int)(idx % per), hk = c / (a.dh / 4), d = c % (a.dh / 4) * 4;
    if (!a.zero_rest && (row < pa_bound(a.ends_k, 1, a.B, a.Tk) || row >= pa_bound(a.ends_k, a.B + 1, a.B, a.Tk))) return;
    const long long step = (long long)a.Tk * a.Hk * a.dh;
    const float* p = a.dkv_part + idx * 4;
    f32x4 k = {0.f, 0.f, 0.f, 0.f}, v = k;
    for (int s = 0; s < a.splits; ++s) {
        k += *(const f32x4*)(p + s * step);
        v += *(const f32x4*)(p + (a.splits + s) * step);
    }
    v4 ko, vo;
#pragma unroll
    for (int j = 0; j < 4; ++j) { ko[j] = (T)(k[j] * a.scale); vo[j] = (T)v[j]; }
    *(v4*)((T*)a.dk.p + row * a.dk.row + hk * a.dk.head + d) = ko;
    *(v4*)((T*)a.dv.p + row * a.dv.row + hk * a.dv.head + d) = vo;
}

// ================================================================================================================================
// launch
// ================================================================================================================================
namespace {
constexpr int PA_MAX_FAR = 1024;
constexpr size_t PA_DIAGONALS = (4 * 32 * 17 + 256) * 4;      // four tiles, and what is read past the last

int pa_launch(void (*kernel)(const PaArgs), dim3 grid, int threads, size_t lds, const PaArgs& a, hipStream_t st) {
    if (lds > 64 * 1024 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) {
        ddpm_set_error("packed_attention: cannot reserve %zu bytes of LDS", lds);
        return DDPM_EHIP;
    }
    hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, st, a);
    return ddpm_check_launch("packed_attention");
}

template <typename T, int DHP, bool BIAS>
int pa_launch_fwd(const PaArgs& a, hipStream_t st) {
    return pa_launch(BIAS && a.o32 ? pa_fwd_kernel<T, DHP, BIAS, BIAS> : pa_fwd_kernel<T, DHP, BIAS, false>, dim3((unsigned)(a.slots * a.H)), 256, 4 * PaTile<DHP>::BYTES + (BIAS ? (2 * a.far + 1) * 4 : 0), a, st);
}

template <typename T, int DHP, bool BIAS>
int pa_launch_bwd(PaArgs a, float* dtable, hipStream_t st) {
    const size_t width = (2 * a.far + 1) * 4;
    if (a.Tq > 0) {
        if (const int rc = pa_launch(pa_bwd_dq_kernel<T, DHP, BIAS>, dim3((unsigned)(a.slots * a.H)), 256, 4 * PaTile<DHP>::BYTES + (BIAS ? (a.dtable_part ? 5 * width + PA_DIAGONALS : width) : 0), a, st)) return rc;
    }
    if (a.dtable_part)
        hipLaunchKernelGGL(pa_dtable_kernel, dim3((unsigned)a.H), dim3(256), 0, st, a.dtable_part, a.Tq > 0 ? a.slots : 0, a.H, a.buckets, dtable);
    constexpr int rows = DHP == 128 ? 32 : PA_TILE;
    a.slots = a.Tk / PA_ROWS + a.B + 2;
    if (a.Tk == 0) return ddpm_check_launch("packed_attention_backward");
    if (const int rc = pa_launch(pa_bwd_dkv_kernel<T, DHP, BIAS>, dim3((unsigned)(a.slots * a.Hk * a.splits)), 256, rows * (4 * PaTile<DHP>::RB + 16) + (BIAS ? (width + 15) / 16 * 16 : 0) + (DHP == 128 ? PA_ROWS * PaTile<DHP>::RB : 0), a, st)) return rc;
    if (a.splits > 1) {
        const long long n = (long long)a.Tk * a.Hk * (a.dh / 4);
        hipLaunchKernelGGL(pa_dkv_join_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    }
    return ddpm_check_launch("packed_attention_backward");
}

// How many workgroups share the queries of 128 keys.  The host knows sizes, not lengths: `groups` of keys, and on average `steps` tiles of
// queries for each.  Two workgroups fit on a CU, and more than one for each of the 512 places evens them out; but each share is written and
// read once more in 32 bits, and begins with k, v.  Backward pass in us, one share against the rule's:
//   336 groups of 74 steps (causal, 128 wide)  503 / 317 (3)      544 of 256 (causal, 128 wide)  1220 / 966 (2)     112 of 44 (causal, 64 wide)  138 / 66 (7)
//   18 of 16 (64 wide)                          73 / 30 (8)       268 of 128 (64 wide)            379 / 307 (3)
// and where it leaves one, against two:  512 of 19 (64 wide) 118 / 136,  176 of 8 (causal, 64 wide) 33 / 38,  4288 of 64 (causal, 128 wide) 2050 / 2530.
int pa_splits(const ddpm_packed_attn_desc* d) {
    const long long groups = (long long)(d->Tk / PA_ROWS + d->B + 2) * d->Hk, steps = (long long)d->Tq / PA_TILE * (d->H / d->Hk) / (d->B > 0 ? d->B : 1);
    const long long most = steps / (groups >= 128 ? 16 : 2);               // (half of the card idle: even short shares pay)
    long long z = (700 + groups - 1) / groups;
    z = z < most ? z : most;
    return z < 1 ? 1 : z > 8 ? 8 : (int)z;
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
    // (a launch is limited to 2^32 - 1 threads)
    DDPM_REQUIRE((int64_t)(d->Tq / PA_ROWS + d->B + 2) * d->H < (1ll << 24) && (int64_t)(d->Tk / PA_ROWS + d->B + 2) * d->Hk < (1ll << 24), "packed_attention: too many workgroups");
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
        DDPM_REQUIRE(d->Tk == 0 || pa_splits(d) == 1 || d->dkv_part, "packed_attention: backward of these sizes needs the workspace dkv_part");
        DDPM_REQUIRE(!d->dtable || d->dtable_part, "packed_attention: the bias's gradient needs the workspace dtable_part");
    }
    a.o32 = d->o32; a.lse = d->lse; a.dsum = d->dsum;
    a.ends_q = d->ends_q; a.ends_k = d->ends_k;
    a.table = d->table; a.bucket_of = d->bucket_of; a.buckets = d->buckets; a.far = d->table ? d->far : 0;
    a.dtable_part = bwd && d->dtable ? d->dtable_part : nullptr;
    a.splits = bwd ? pa_splits(d) : 1;
    a.dkv_part = a.splits > 1 ? d->dkv_part : nullptr;
    a.Tq = d->Tq; a.Tk = d->Tk; a.B = d->B; a.H = d->H; a.Hk = d->Hk; a.dh = d->dh; a.causal = d->causal; a.zero_rest = d->zero_rest;
    a.slots = d->Tq / PA_ROWS + d->B + 2;
    a.scale = d->scale;
    a.scale2 = d->scale * 1.4426950408889634f;
    return DDPM_OK;
}
}  // namespace

extern "C" int ddpm_packed_attn_slots(int Tq, int B) { return Tq / PA_ROWS + B + 2; }
extern "C" int64_t ddpm_packed_attn_dkv_floats(const ddpm_packed_attn_desc* d) {
    // (sizes that the backward pass refuses need nothing)
    const bool sizes = d && d->H > 0 && d->Hk > 0 && d->Tq >= 0 && d->Tk >= 0 && d->B >= 0 && d->Tq < (1 << 30) && d->Tk < (1 << 30) && d->B < (1 << 24);
    const int splits = sizes ? pa_splits(d) : 1;
    return splits > 1 ? 2ll * splits * d->Tk * d->Hk * d->dh : 0;
}

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
