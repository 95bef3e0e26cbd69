// Pieces shared by the attention kernels that work on whole tiles of fp16 tokens (prompt attention, wide trees): the score
// modifiers, the LDS layout of a tile and the two matrix products on it.
//
// Everything is computed transposed: S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16_f16.  A lane then owns one
// query row (column lane & 31 of the accumulators) and half of a tile's tokens, so the softmax of a row is arithmetic
// inside a lane plus one exchange with lane ^ 32, and the probabilities leave the first product in the very lanes in which
// the second one wants them: accumulator register r of half h holds token 8 (r / 4) + 4 h + r % 4, and since a contraction
// index may be numbered at will, the second product takes its tokens in that order.
#pragma once

#include "akv_common.h"

namespace akv {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4v __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kNegInf = -__builtin_inff();

__device__ __forceinline__ f16x8 as_f16x8(u32x4 w) { return __builtin_bit_cast(f16x8, w); }
__device__ __forceinline__ u32 pack_f16(float a, float b) {   // round to nearest even
    const f32x2 f = {a, b};
    return __builtin_bit_cast(u32, __builtin_convertvector(f, f16x2v));
}

// Maximum / sum over a lane and the lane 32 away (the other half of the wave), the same in both.
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// tanh in 32 bits.  |y| <= 0.6: an odd polynomial through y^9, fitted to tanh there (largest error 2.8e-8, below half a step of
// tanh(0.6)); 1 - 2 / (exp(2 y) + 1) would lose small arguments to cancellation, and a capped score is cap * tanh, so what
// is lost is multiplied by the cap.  Beyond: that form, from the hardware's 2^x and reciprocal.
constexpr float kTanhNear = 0.6f;
__device__ __forceinline__ float tanh_near(float y) {
    const float z = y * y;
    float p = fmaf(z, 0.015319169f, -0.051994310f);
    p = fmaf(z, p, 0.13308098f);
    p = fmaf(z, p, -0.33332248f);
    return fmaf(y * z, p, y);
}
__device__ __forceinline__ float tanh_f32(float y) {
    const float e = __builtin_amdgcn_exp2f(y * (2.f * kLog2e));
    float far = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
    asm volatile("" : "+v"(far));      // both forms in straight code: a branch per score would cost more
    return fabsf(y) <= kTanhNear ? tanh_near(y) : far;     // (not-a-number: far, which is not one either)
}

// What a raw product q . k goes through, in units of log2 e (so that the softmax takes 2^x):
//   no cap: x = raw * c0;  cap: x = c1 * tanh(raw * c0);  then x -= slope * |distance|.
struct ScoreForm {
    float c0, c1;
    float near, n1, n2, n3;      // |raw| <= near: x = c1 c0 raw (1 + n1 raw^2 + n2 raw^4 + n3 raw^6)
};
__host__ __device__ __forceinline__ ScoreForm score_form(float scale, float cap) {
    ScoreForm f = {scale * kLog2e, 1.f, -1.f, 0.f, 0.f, 0.f};
    if (cap > 0.f) {
        f.c0 = scale / cap;
        f.c1 = cap * kLog2e;
        // an odd polynomial through the seventh power, fitted to tanh on |y| <= 0.4 (largest error 2.8e-8, half a step of tanh there), its
        // coefficients for raw instead of y = raw * c0; powers that fp32 does not hold: no such range
        const float z = f.c0 * f.c0;
        if (f.c0 > 1e-5f && f.c0 < 1e5f) f = {f.c0, f.c1, 0.4f / f.c0, -0.333313877f * z, 0.132687496f * z * z, -0.0474229918f * z * z * z};
    }
    return f;
}
template <bool CAP>
__device__ __forceinline__ float modified(float raw, const ScoreForm &f) {
    if constexpr (CAP) return f.c1 * tanh_f32(raw * f.c0);
    return raw * f.c0;
}
// The same for a register block of a wave, up to the factor that is returned (a softmax multiplies it in where it subtracts the
// maximum).  Capped scores are mostly far below their cap: where all of the wave's are, the polynomial alone is evaluated (5
// instructions a score instead of 20, two of them at a quarter of the rate).
template <bool CAP, int NB>
__device__ __forceinline__ float modify_block(f32x16 (&x)[NB], const ScoreForm &f) {
    if constexpr (!CAP) return f.c0;
    float most = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(x[b][r]));
    if (__all(most <= f.near)) {      // (fmaxf passes over not-a-number; the polynomial hands it on)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float z = x[b][r] * x[b][r];
                x[b][r] *= fmaf(z, fmaf(z, fmaf(z, f.n3, f.n2), f.n1), 1.f);
                if (r % 8 == 7) __builtin_amdgcn_sched_barrier(0);
            }
        return f.c0 * f.c1;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[b][r] = tanh_f32(x[b][r] * f.c0);
            if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);      // (four at a time: all 32 at once need more registers than there are)
        }
    return f.c1;
}

// ---- a tile of BN tokens x D channels in LDS, fp16, token-major ------------------------------------------------------------
// 16-byte chunk c of row r lies at chunk c ^ swizzle(r): the lanes of one LDS access then spread over all banks, both for
// the K operand (8 consecutive rows, one chunk) and for the transposed V operand (4 consecutive rows, 64 bytes each).
template <int D>
__device__ __forceinline__ int tile_swizzle(int row) {
    if constexpr (D == 64) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);   // two rows per 256 bytes of banks
    return (row & 3) << 2 | ((row >> 2) & 3);
}
template <int D>
__device__ __forceinline__ int tile_byte(int row, int chunk) {
    return row * (D * 2) + ((chunk ^ tile_swizzle<D>(row)) << 4);
}

// 16 bytes a lane from memory straight into LDS, lane l's at lds_base + 16 l (lds_base: the same in all lanes); nothing passes
// through registers.  The compiler does not see these loads: wait_tile() before what they bring is read.  M0 holds the LDS address, and
// one wait state has to lie between its write and the load; inside inline assembly the compiler does not put it there.
__device__ __forceinline__ u32 lds_address(const void *p) { return (u32)(uintptr_t)(__attribute__((address_space(3))) const void *)p; }
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, u32 lds_base, int byte_off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(__builtin_amdgcn_readfirstlane((int)lds_base)), "v"(byte_off), "s"(r)
                 : "memory", "m0");
}
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// All of this wave's loads have arrived and its LDS reads are done, and so are the other waves'.
__device__ __forceinline__ void wait_tile() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

typedef __attribute__((address_space(3))) s16x4 *lds_s16x4_ptr;

// Where a lane reads its operands in a tile: the part of the addresses that depends on the lane, so that what differs from read
// to read is a constant (rows 16 apart lie alike) or one exclusive-or.
template <int D>
struct LaneBytes {
    int k;                 // K operand, step 0; step ks: k ^ (ks << 5)
    int v[2];              // V^T operand, channels 0 .. 31, first and second group of four tokens; block cb: v ^ (cb << 6)
    __device__ __forceinline__ LaneBytes() {
        const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5;
        k = tile_byte<D>(row, half);
        const int vr = 4 * half + ((lane & 15) >> 2), chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), in_chunk = (lane & 1) * 8;
        v[0] = tile_byte<D>(vr, chunk) + in_chunk;
        v[1] = tile_byte<D>(vr + 8, chunk) + in_chunk;
    }
    // Once per tile: what is derived from these is worked out again (one instruction a read) instead of being kept in registers.
    __device__ __forceinline__ void pin() { asm volatile("" : "+v"(k), "+v"(v[0]), "+v"(v[1])); }
};

// S^T of one tile: acc[tb] = K rows 32 tb .. 32 tb + 31 times the wave's 32 query rows.  qf[ks]: channels 16 ks + 8 half ..
template <int D, int BN>
__device__ __forceinline__ void tile_scores(f32x16 (&acc)[BN / 32], const uint8_t *k_tile, const LaneBytes<D> &at, const f16x8 (&qf)[D / 16]) {
#pragma unroll
    for (int tb = 0; tb < BN / 32; ++tb)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[tb][r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        const uint8_t *kp = k_tile + (at.k ^ (ks << 5));
#pragma unroll
        for (int tb = 0; tb < BN / 32; ++tb)
            acc[tb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const f16x8 *>(kp + tb * 32 * D * 2), qf[ks], acc[tb], 0, 0, 0);
        if (ks % 4 == 3) __builtin_amdgcn_sched_barrier(0);     // (operands of four steps in flight; all of them would not fit beside the sums)
    }
}

// The V^T operand for channels 32 cb .. + 31 and the 16 tokens whose probabilities are registers 8 s .. 8 s + 7 of block tb:
// two transposing reads of four tokens each (lane group of 16: row r from the lanes 4 r .. 4 r + 3, column = lane).
template <int D>
__device__ __forceinline__ f16x8 tile_v_operand(const uint8_t *v_tile, const LaneBytes<D> &at, int cb, int tb, int s) {
    const int rows = (tb * 32 + s * 16) * D * 2;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(v_tile + (at.v[0] ^ (cb << 6)) + rows));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(v_tile + (at.v[1] ^ (cb << 6)) + rows));
    return __builtin_bit_cast(f16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// ---- infinite or undefined values in a V tile that some rows see only in part ----------------------------------------------------
// A hidden token's probability is zero, but zero times such a value is undefined.  On a tile at the edge of what some row of the
// workgroup sees, the waves look through the values first (a share each).  Where one is not finite (rare) what these values do
// is noted apart: a row that sees +inf (or not-a-number) in a channel gets +inf added to its output there in the end, one that sees
// -inf (or not-a-number) -inf; then they are zeroed in LDS and the tile goes the usual way.
template <int D>
struct OddValues {
    u32 hit[2][D / 64] = {};      // [+inf, -inf]: bit 16 (cb % 2) + r of word cb / 2: this lane's row, channel of register r of block cb
    __device__ __forceinline__ bool any() const {
        u32 x = 0;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < D / 64; ++i) x |= hit[s][i];
        return __any(x != 0);
    }
    __device__ __forceinline__ void add(f32x16 (&o)[D / 32]) const {
#pragma unroll
        for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const u32 bit = 1u << (16 * (cb & 1) + r);
                o[cb][r] += (hit[0][cb >> 1] & bit ? __builtin_inff() : 0.f) - (hit[1][cb >> 1] & bit ? __builtin_inff() : 0.f);
            }
    }
};

// This wave's share of the tile (THREADS threads look through it, this is number tid): does it hold such a value?
template <int D, int BN, int THREADS>
__device__ __forceinline__ bool share_nonfinite(const uint8_t *v_tile, int tid) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 most = {0, 0};
#pragma unroll
    for (int c = 0; c < BN * D / (8 * THREADS); ++c) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(v_tile + (c * THREADS + tid) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
    }
    return __any(most.x >= 0x7C00 || most.y >= 0x7C00);
}
__device__ __forceinline__ f16x8 zero_nonfinite(f16x8 v) {
    u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u32 x = w[i];
        x = (x & 0x7C00u) == 0x7C00u ? x & 0xFFFF0000u : x;
        x = (x & 0x7C000000u) == 0x7C000000u ? x & 0x0000FFFFu : x;
        w[i] = x;
    }
    return __builtin_bit_cast(f16x8, w);
}

// O^T += V^T P^T for one tile.  p[tb][s]: the probabilities as packed above.
template <int D, int BN>
__device__ __forceinline__ void tile_output(f32x16 (&o)[D / 32], const uint8_t *v_tile, const LaneBytes<D> &at, const f16x8 (&p)[BN / 32][2]) {
#pragma unroll
    for (int tb = 0; tb < BN / 32; ++tb)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int cb = 0; cb < D / 32; ++cb)
                o[cb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(tile_v_operand<D>(v_tile, at, cb, tb, s), p[tb][s], o[cb], 0, 0, 0);
}

// seen: bit 16 tb + r says that this lane's row sees the token of register r of block tb.
template <int D, int BN>
__device__ __forceinline__ void note_nonfinite(OddValues<D> &odd, const uint8_t *v_tile, const LaneBytes<D> &at, u32 seen) {
    const u32 one = 0x3C00u;      // 1 in fp16
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
        for (int sign = 0; sign < 2; ++sign) {
            f32x16 hits;          // how many +inf / -inf (not-a-number: both) each row sees in each channel
#pragma unroll
            for (int r = 0; r < 16; ++r) hits[r] = 0.f;
#pragma unroll 1
            for (int ts = 0; ts < BN / 16; ++ts) {
                const u32x4 v = __builtin_bit_cast(u32x4, tile_v_operand<D>(v_tile, at, cb, ts >> 1, ts & 1));
                u32x4 is, sees;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u32 lo = v[i] & 0xFFFFu, hi = v[i] >> 16;
                    const bool a = (lo & 0x7FFFu) > 0x7C00u || lo == (sign ? 0xFC00u : 0x7C00u), c = (hi & 0x7FFFu) > 0x7C00u || hi == (sign ? 0xFC00u : 0x7C00u);
                    is[i] = (a ? one : 0u) | (c ? one << 16 : 0u);
                    const u32 bits = seen >> (8 * ts + 2 * i);
                    sees[i] = (bits & 1u ? one : 0u) | (bits & 2u ? one << 16 : 0u);
                }
                hits = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_f16x8(is), as_f16x8(sees), hits, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) odd.hit[sign][cb >> 1] |= hits[r] > 0.f ? 1u << (16 * (cb & 1) + r) : 0u;
            asm volatile("" : "+v"(odd.hit[sign][cb >> 1]));      // now: not with the counts of all eight loops in registers
        }
}
template <int D, int BN, int THREADS>
__device__ __forceinline__ void zero_nonfinite_tile(uint8_t *v_tile, int tid) {
#pragma unroll 1
    for (int c = 0; c < BN * D / (8 * THREADS); ++c) {
        f16x8 *w = reinterpret_cast<f16x8 *>(v_tile + (c * THREADS + tid) * 16);
        *w = zero_nonfinite(*w);
    }
}

// Running softmax state of the wave's 32 rows (a row's two lanes hold the same m and their own part of l).
struct RowState {
    float m = kNegInf;   // maximum the sums are relative to (units of log2 e)
    float l = 0.f;       // this lane's share of the sum
};

// Probabilities are formed as 2^(score - m + kLift), m a running maximum that is raised when a row's has grown by more than kGrown: at most
// 2^15, which fp16 holds, and the row's largest at least 2^kLift.  Rounded to fp16 a probability is off by 2^-11 of itself or, where fp16 is
// subnormal, by 2^-25, which is 2^-32 of the row's largest; without the lift it is 2^-25 of it, and where one token takes the weight and its
// value is small, the many small terms beside it are lost (32768 tokens 16 / 17 / 20 natural units below one of value zero: relative error
// 1.0e-2 / 0.11 / 0.25 without, 1.5e-4 / 2.0e-4 / 3.2e-4 with it).  Its cost is below what two runs differ by (prompts of 8192 tokens 323 to
// 327 us without, 319 to 333 with it).  Sums and outputs carry the same factor, which a division takes out; the logarithm of a sum subtracts it.
constexpr float kGrown = 8.f, kLift = 7.f;

// Scores factor * x[tb][r] + shift (factor > 0; units of log2 e; x -inf where hidden) -> packed probabilities 2^(score - m + kLift); rescales l
// and o when the maximum grew by more than kGrown, which after the first tiles of a row is rare.
template <int D, int BN>
__device__ __forceinline__ void tile_softmax(f32x16 (&x)[BN / 32], float factor, float shift, RowState &st, f32x16 (&o)[D / 32], f16x8 (&p)[BN / 32][2]) {
    float mx = x[0][0];
#pragma unroll
    for (int tb = 0; tb < BN / 32; ++tb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, x[tb][r]);
    mx = halves_max(fmaf(mx, factor, shift));
    if (__any(mx > st.m + kGrown)) {     // (m = -inf: any finite maximum)
        const float m_new = fmaxf(st.m, mx);
        const float alpha = st.m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(st.m - m_new);
        st.m = m_new;
        st.l *= alpha;
#pragma unroll
        for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[cb][r] *= alpha;
    }
    const float less = shift - (st.m == kNegInf ? 0.f : st.m) + kLift;
    float sum = 0.f;
#pragma unroll
    for (int tb = 0; tb < BN / 32; ++tb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[tb][r] = __builtin_amdgcn_exp2f(fmaf(x[tb][r], factor, less));
            sum += x[tb][r];
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_f16(x[tb][8 * s + 2 * i], x[tb][8 * s + 2 * i + 1]);
            p[tb][s] = as_f16x8(w);
        }
    }
    st.l += sum;
}

// Whether two stretches of memory share a byte (what is written has to lie apart from what other workgroups still read).
inline bool share_memory(const void *a, int64_t bytes_a, const void *b, int64_t bytes_b) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + (uintptr_t)bytes_b && y < x + (uintptr_t)bytes_a;
}
// Bytes from the first to the last of fp32 rows [B, H, n].
inline int64_t rows_span(int64_t B, int64_t H, int64_t n, int64_t stride_b, int64_t stride_h) { return 4 * ((B - 1) * stride_b + (H - 1) * stride_h + n); }
// Whether such rows lie apart, sequence by sequence or head by head: they are added to without atomics.
inline bool rows_apart(int64_t B, int64_t H, int64_t n, int64_t stride_b, int64_t stride_h) {
    return ((H == 1 || stride_h >= n) && (B == 1 || stride_b >= (H - 1) * stride_h + n)) ||
           ((B == 1 || stride_b >= n) && (H == 1 || stride_h >= (B - 1) * stride_b + n));
}

int check_layer(const akv_cache_layer *c, const char *what);   // of a cache layer's descriptor: AKV_OK or the error

}  // namespace akv
