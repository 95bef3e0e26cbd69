// Attention of a tree of drafted tokens over the split-plane cache, and the commit of the drafts that were accepted.
//
// T drafted tokens per sequence attend to the whole cache (planes and rest buffer, every plane: a row of planes is needed
// at full precision as soon as one of the T x G query rows of a KV head needs it) and to the drafts in their ancestors'
// bit mask.  The cache does not change until tree_commit appends the accepted path.
#include "akv_attention.h"

namespace akv {

typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int kRest = 64;       // tokens of the rest buffer

struct TreeArgs {
    akv_cache_layer c;
    const uint8_t *q, *k, *v;             // fp16 [B, T, Hq | Hkv, D]
    const unsigned long long *anc;        // [T] or [B, T]
    int anc_stride;                       // T or 0
    const float *slopes;
    uint8_t *out;
    float *parts;                         // [B * Hkv, splits, rows] x {D sums}, then the same x {m, l}
    int T, Hq, G, rows;                   // rows = T * G
    int plane_splits, tiles_per_split, splits;
    ScoreForm form;
};

// Cached tokens of a sequence, kept inside the planes whatever the device holds.
__device__ __forceinline__ int cached_tokens(const TreeArgs &a, int b) { return max(0, min(a.c.seq_lens[b], a.c.max_seq_len)); }

// acc[t] += K (tokens) x Q^T for one step of 32 channels.  A lane (m, kg) holds 8 channels x TPL tokens of token set m; operand t
// is token t of every set, so no value leaves its lane.
template <int TPL>
struct KStep {
    u32 h[8][TPL / 4], m[8][TPL / 8], l[8][TPL / 8];
};

template <int N>
__device__ __forceinline__ void load_words(u32 (&w)[N], __amdgpu_buffer_rsrc_t r, int off) {
    if constexpr (N == 1) w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, kStream);
    if constexpr (N == 2) {
        const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, kStream);
        w[0] = x.x;
        w[1] = x.y;
    }
    if constexpr (N == 4) {
        const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, kStream);
        w[0] = x.x;
        w[1] = x.y;
        w[2] = x.z;
        w[3] = x.w;
    }
}

// 16-bit values of elements 0,2 / 1,3 / 4,6 / 5,7 of 8 elements (high bytes Ha, Hb; nibbles M, L)
__device__ __forceinline__ void rebuild8(u32 Ha, u32 Hb, u32 M, u32 L, u32 &w02, u32 &w13, u32 &w46, u32 &w57) {
    u32 E, O;
    split_even_odd(M, L, E, O);
    w02 = __builtin_amdgcn_perm(Ha, E, 0x06010400u);
    w13 = __builtin_amdgcn_perm(Ha, O, 0x07010500u);
    w46 = __builtin_amdgcn_perm(Hb, E, 0x06030402u);
    w57 = __builtin_amdgcn_perm(Hb, O, 0x07030502u);
}
__device__ __forceinline__ u32 low_halves(u32 a, u32 b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ u32 high_halves(u32 a, u32 b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// 8 x 8 block of halves held as w[i] (i: index of the pair partner list) -> operand dwords.  in: for each of 8 rows i the words
// {02, 13, 46, 57} of 8 columns; out[c][p]: column c, rows 2 p and 2 p + 1.
__device__ __forceinline__ void transpose8(const u32 (&w)[8][4], u32 (&out)[8][4]) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const u32 (&a)[4] = w[2 * p], (&b)[4] = w[2 * p + 1];
        out[0][p] = low_halves(a[0], b[0]);
        out[2][p] = high_halves(a[0], b[0]);
        out[1][p] = low_halves(a[1], b[1]);
        out[3][p] = high_halves(a[1], b[1]);
        out[4][p] = low_halves(a[2], b[2]);
        out[6][p] = high_halves(a[2], b[2]);
        out[5][p] = low_halves(a[3], b[3]);
        out[7][p] = high_halves(a[3], b[3]);
    }
}
__device__ __forceinline__ f16x8 operand(const u32 (&w)[4]) { return as_f16x8(u32x4{w[0], w[1], w[2], w[3]}); }

// Over the four lanes n, n + 16, n + 32, n + 48 of a column.
__device__ __forceinline__ float column_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float column_sum(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return halves_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// One wave's running state for NT x 16 query rows: a lane owns column n = lane & 15 of every tile of rows.
template <int D, int NT>
struct Rows {
    static constexpr int CPL = D / 16;        // channels of a lane's set: channel CPL * (4 kg + r) + j
    f16x8 q[NT][D / 32];
    f32x4 o[NT][CPL];
    float m[NT], l[NT];
    unsigned long long anc[NT];
    int pos[NT];                              // the row's position
    float neg_slope[NT];
};

// x[i] (units of log2 e, -inf where hidden), N values of one column per lane -> probabilities, state and outputs rescaled.
template <int D, int NT, int N>
__device__ __forceinline__ void rows_softmax(float (&x)[N], Rows<D, NT> &s, int nt) {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mx = fmaxf(mx, x[i]);
    mx = column_max(mx);
    if (__any(mx > s.m[nt] + 8.f)) {
        const float m_new = fmaxf(s.m[nt], mx);
        const float alpha = s.m[nt] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(s.m[nt] - m_new);
        s.m[nt] = m_new;
        s.l[nt] *= alpha;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) s.o[nt][j] *= alpha;
    }
    const float m = s.m[nt] == kNegInf ? 0.f : s.m[nt];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = __builtin_amdgcn_exp2f(x[i] - m);
        sum += x[i];
    }
    s.l[nt] += sum;
}

// One tile of 16 * TPL tokens of the planes starting at token j0 (a multiple of 64), n_valid of them in the planes (a multiple of 64).
template <int D, int KB, int TPL, int NT, bool CAP, bool ALIBI>
__device__ __forceinline__ void plane_tile(const TreeArgs &a, Rows<D, NT> &s, int64_t bh, int j0, int n_valid) {
    constexpr int CPL = D / 16;
    const int lane = threadIdx.x & 63, m = lane & 15, kg = lane >> 4;
    const bool k_in = m * TPL < n_valid, v_in = kg * 4 * TPL < n_valid;
    f32x4 acc[NT][TPL];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < TPL; ++t) acc[nt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    {
        const int64_t blk = bh * a.c.n_max_blocks + j0 / KB;
        const int blocks = KB == 64 ? (n_valid + 63) / 64 : 1, tok0 = j0 % KB + m * TPL;
        const auto rh = make_rsrc(a.c.k_first_8 + blk * (D * KB), blocks * D * KB);
        const auto rm = make_rsrc(a.c.k_mid_4 + blk * (D * KB / 2), blocks * D * KB / 2);
        const auto rl = make_rsrc(a.c.k_last_4 + blk * (D * KB / 2), blocks * D * KB / 2);
        const int base = KB == 64 ? (tok0 / 64) * (D * 64) + tok0 % 64 : tok0;
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
            KStep<TPL> w;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int off = base + (ks * 32 + kg * 8 + i) * KB;
                load_words(w.h[i], rh, k_in ? off : kSkip);
                load_words(w.m[i], rm, k_in ? off >> 1 : kSkip);
                load_words(w.l[i], rl, k_in ? off >> 1 : kSkip);
            }
#pragma unroll
            for (int g = 0; g < TPL / 8; ++g) {
                u32 in[8][4], op[8][4];
#pragma unroll
                for (int i = 0; i < 8; ++i) rebuild8(w.h[i][2 * g], w.h[i][2 * g + 1], w.m[i][g], w.l[i][g], in[i][0], in[i][1], in[i][2], in[i][3]);
                transpose8(in, op);
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        acc[nt][8 * g + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand(op[t]), s.q[nt][ks], acc[nt][8 * g + t], 0, 0, 0);
            }
        }
    }
    // lane (n, kg): token TPL * (4 kg + r) + t of the tile in acc[t][r]
    u32 p[NT][TPL * 4 / 8][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float x[4 * TPL];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int t = 0; t < TPL; ++t) {
                float y = modified<CAP>(acc[nt][t][r], a.form);
                if constexpr (ALIBI) y = fmaf(s.neg_slope[nt], fabsf((float)(s.pos[nt] - (j0 + TPL * (4 * kg + r) + t))), y);
                x[r * TPL + t] = v_in ? y : kNegInf;
            }
        rows_softmax<D, NT, 4 * TPL>(x, s, nt);
#pragma unroll
        for (int st = 0; st < TPL / 2; ++st)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[nt][st][i] = pack_f16(x[8 * st + 2 * i], x[8 * st + 2 * i + 1]);
    }
    {
        // eight consecutive tokens per step and lane, channels CPL * m .. of each
        const int64_t row0 = bh * a.c.max_seq_len + j0;
        const auto rh = make_rsrc(a.c.v_first_8 + row0 * D, n_valid * D);
        const auto rm = make_rsrc(a.c.v_mid_4 + row0 * (D / 2), n_valid * D / 2);
        const auto rl = make_rsrc(a.c.v_last_4 + row0 * (D / 2), n_valid * D / 2);
#pragma unroll
        for (int st = 0; st < TPL / 2; ++st) {
            u32 h[8][(CPL + 3) / 4], md[8][(CPL + 7) / 8], ls[8][(CPL + 7) / 8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int off = (kg * 4 * TPL + 8 * st + i) * D + CPL * m;
                load_words(h[i], rh, v_in ? off : kSkip);
                if constexpr (CPL == 4) {
                    md[i][0] = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rm, v_in ? off >> 1 : kSkip, 0, kStream);
                    ls[i][0] = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rl, v_in ? off >> 1 : kSkip, 0, kStream);
                } else {
                    load_words(md[i], rm, v_in ? off >> 1 : kSkip);
                    load_words(ls[i], rl, v_in ? off >> 1 : kSkip);
                }
            }
#pragma unroll
            for (int g = 0; g < (CPL + 7) / 8; ++g) {
                u32 in[8][4], op[8][4];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    rebuild8(h[i][2 * g], CPL == 4 ? 0u : h[i][(2 * g + 1) % ((CPL + 3) / 4)], md[i][g], ls[i][g], in[i][0], in[i][1], in[i][2], in[i][3]);
                transpose8(in, op);
#pragma unroll
                for (int c = 0; c < (CPL < 8 ? CPL : 8); ++c)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        s.o[nt][8 * g + c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand(op[c]), operand(p[nt][st]), s.o[nt][8 * g + c], 0, 0, 0);
            }
        }
    }
}

// 32 tokens of the tail: the rest buffer's n_rest tokens, then the T drafts; u0: first token of this tile.
template <int D, int NT, bool CAP, bool ALIBI>
__device__ __forceinline__ void tail_tile(const TreeArgs &a, Rows<D, NT> &s, int b, int hkv, int u0, int n_rest, int n) {
    constexpr int CPL = D / 16;
    const int lane = threadIdx.x & 63, m = lane & 15, kg = lane >> 4, H = a.c.n_kv_heads, total = n_rest + a.T;
    const uint8_t *rk = a.c.restk + ((int64_t)b * kRest * H + hkv) * (D * 2), *rv = a.c.restv + ((int64_t)b * kRest * H + hkv) * (D * 2);
    const uint8_t *dk = a.k + ((int64_t)b * a.T * H + hkv) * (D * 2), *dv = a.v + ((int64_t)b * a.T * H + hkv) * (D * 2);
    const int64_t row_bytes = (int64_t)H * D * 2;
    const auto k_row = [&](int u) { return u < n_rest ? rk + u * row_bytes : dk + (min(u, total - 1) - n_rest) * row_bytes; };
    const auto v_row = [&](int u) { return u < n_rest ? rv + u * row_bytes : dv + (min(u, total - 1) - n_rest) * row_bytes; };
    f32x4 acc[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint8_t *kp = k_row(u0 + 16 * t + m);
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
            const f16x8 w = *reinterpret_cast<const f16x8 *>(kp + (ks * 32 + kg * 8) * 2);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, s.q[nt][ks], acc[nt][t], 0, 0, 0);
        }
    }
    // lane (n, kg): token u0 + 16 t + 4 kg + r in acc[t][r]
    const unsigned long long *anc = a.anc + (int64_t)b * a.anc_stride;
    const auto visible = [&](int nt, int u) { return u < n_rest || (u < total && ((s.anc[nt] >> (u - n_rest)) & 1)); };
    u32 p[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float x[8];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int u = u0 + 16 * t + 4 * kg + r;
                float y = modified<CAP>(acc[nt][t][r], a.form);
                if constexpr (ALIBI) {
                    const int d = min(max(u - n_rest, 0), a.T - 1);
                    const int at = u < n_rest ? n - n_rest + u : n + __popcll(anc[d] & ~(1ull << d));
                    y = fmaf(s.neg_slope[nt], fabsf((float)(s.pos[nt] - at)), y);
                }
                x[4 * t + r] = visible(nt, u) ? y : kNegInf;
            }
        rows_softmax<D, NT, 8>(x, s, nt);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[nt][i] = pack_f16(x[2 * i], x[2 * i + 1]);
    }
    bool bad = false;
#pragma unroll
    for (int g = 0; g < (CPL + 7) / 8; ++g) {
        u32 in[8][4], op[8][4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int u = u0 + 16 * (i >> 2) + 4 * kg + (i & 3);
            const uint8_t *vp = v_row(u) + (CPL * m + 8 * g) * 2;
            const u32 w0 = *reinterpret_cast<const u32 *>(vp), w1 = *reinterpret_cast<const u32 *>(vp + 4);
            u32 w2 = 0, w3 = 0;
            if constexpr (CPL >= 8) {
                w2 = *reinterpret_cast<const u32 *>(vp + 8);
                w3 = *reinterpret_cast<const u32 *>(vp + 12);
            }
            in[i][0] = low_halves(w0, w1);
            in[i][1] = high_halves(w0, w1);
            in[i][2] = low_halves(w2, w3);
            in[i][3] = high_halves(w2, w3);
        }
        transpose8(in, op);
#pragma unroll
        for (int c = 0; c < (CPL < 8 ? CPL : 8); ++c) {
            bad |= any_nonfinite(operand(op[c]));
            const f16x8 w = zero_nonfinite(operand(op[c]));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                s.o[nt][8 * g + c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, operand(p[nt]), s.o[nt][8 * g + c], 0, 0, 0);
        }
    }
    if (!__any(bad)) return;
    // infinite or undefined values reach exactly the rows that see their token
#pragma unroll 1
    for (int u = u0; u < min(u0 + 32, total); ++u) {
        const uint8_t *vp = v_row(u);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (!visible(nt, u)) continue;
#pragma unroll
            for (int j = 0; j < CPL; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float f = (float)*reinterpret_cast<const _Float16 *>(vp + (CPL * (4 * kg + r) + j) * 2);
                    if (!(fabsf(f) < __builtin_inff())) s.o[nt][j][r] += f;
                }
        }
    }
}

// grid (splits, Hkv * row groups, B), 256 threads.  Split s < plane_splits: tiles of the planes, one a wave at a time; the last split: the
// rest buffer and the drafts.  The four waves of a workgroup join their rows' sums through LDS and write one partial result.
template <int D, int KB, int TPL, int NT, bool CAP, bool ALIBI>
__global__ __launch_bounds__(256) void tree_kernel(TreeArgs a) {
    constexpr int CPL = D / 16, TOK = 16 * TPL;
    __shared__ float part[4][16][D + 4];
    __shared__ float ms[4][16], ls[4][16];
    const int lane = threadIdx.x & 63, wave = wave_index(), n_col = lane & 15, kg = lane >> 4;
    const int groups = (a.rows + NT * 16 - 1) / (NT * 16);
    const int split = blockIdx.x, hkv = blockIdx.y / groups, rg = blockIdx.y - hkv * groups, b = blockIdx.z;
    const int n = cached_tokens(a, b), flushed = n / kRest * kRest, n_rest = n - flushed;
    const int64_t bh = (int64_t)b * a.c.n_kv_heads + hkv;
    Rows<D, NT> s;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = min(rg * NT * 16 + nt * 16 + n_col, a.rows - 1), g = row / a.T, t = row - g * a.T;
        const uint8_t *qp = a.q + (((int64_t)b * a.T + t) * a.Hq + hkv * a.G + g) * (D * 2);
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) s.q[nt][ks] = *reinterpret_cast<const f16x8 *>(qp + (ks * 32 + kg * 8) * 2);
#pragma unroll
        for (int j = 0; j < CPL; ++j) s.o[nt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        s.m[nt] = kNegInf;
        s.l[nt] = 0.f;
        s.anc[nt] = a.anc[(int64_t)b * a.anc_stride + t];
        s.pos[nt] = n + __popcll(s.anc[nt] & ~(1ull << t));
        s.neg_slope[nt] = ALIBI ? a.slopes[hkv * a.G + g] * -kLog2e : 0.f;
    }
    if (split < a.plane_splits) {
        const int first = split * a.tiles_per_split, end = min(first + a.tiles_per_split, (flushed + TOK - 1) / TOK);
        for (int t = first + wave; t < end; t += 4)
            plane_tile<D, KB, TPL, NT, CAP, ALIBI>(a, s, bh, t * TOK, min(TOK, flushed - t * TOK));
    } else {
        for (int u0 = wave * 32; u0 < n_rest + a.T; u0 += 128) tail_tile<D, NT, CAP, ALIBI>(a, s, b, hkv, u0, n_rest, n);
    }
    float *po = a.parts + (bh * a.splits + split) * (int64_t)a.rows * D;
    float *pm = a.parts + (int64_t)a.c.bsz * a.c.n_kv_heads * a.splits * a.rows * D + (bh * a.splits + split) * (int64_t)a.rows * 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float l = column_sum(s.l[nt]);
        if (kg == 0) {
            ms[wave][n_col] = s.m[nt];
            ls[wave][n_col] = l;
        }
#pragma unroll
        for (int j = 0; j < CPL; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[wave][n_col][CPL * (4 * kg + r) + j] = s.o[nt][j][r];
        __syncthreads();
        for (int id = threadIdx.x; id < 16 * D; id += 256) {
            const int col = id / D, ch = id - col * D, row = rg * NT * 16 + nt * 16 + col;
            const float m = fmaxf(fmaxf(ms[0][col], ms[1][col]), fmaxf(ms[2][col], ms[3][col]));
            float o = 0.f, sum = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = ms[w][col] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(ms[w][col] - m);
                // a wave that saw nothing has sums of zero, unless a value it did see was undefined: then so is the row
                o += part[w][col][ch] * f;
                sum += ls[w][col] * f;
            }
            if (row < a.rows) {
                po[(int64_t)row * D + ch] = o;
                if (ch == 0) {
                    pm[row * 2] = m;
                    pm[row * 2 + 1] = sum;
                }
            }
        }
        if (nt + 1 < NT) __syncthreads();
    }
}

// One workgroup of D threads per query row: joins the splits in order.
template <int D>
__global__ __launch_bounds__(D) void tree_combine_kernel(TreeArgs a) {
    const int row = blockIdx.x, hkv = blockIdx.y, b = blockIdx.z, ch = threadIdx.x;
    const int64_t bh = (int64_t)b * a.c.n_kv_heads + hkv;
    const float *po = a.parts + bh * a.splits * (int64_t)a.rows * D + (int64_t)row * D + ch;
    const float *pm = a.parts + (int64_t)a.c.bsz * a.c.n_kv_heads * a.splits * a.rows * D + bh * a.splits * (int64_t)a.rows * 2 + row * 2;
    float m = kNegInf;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, pm[(int64_t)s * a.rows * 2]);
    float o = 0.f, l = 0.f;
    for (int s = 0; s < a.splits; ++s) {
        const float ms = pm[(int64_t)s * a.rows * 2];
        const float f = ms == kNegInf ? 0.f : __builtin_amdgcn_exp2f(ms - m);
        o = fmaf(po[(int64_t)s * a.rows * D], f, o);
        l = fmaf(pm[(int64_t)s * a.rows * 2 + 1], f, l);
    }
    const float r = l == 0.f ? o : o / l;      // (a row that saw nothing: zero)
    const int g = row / a.T, t = row - g * a.T;
    reinterpret_cast<unsigned short *>(a.out)[(((int64_t)b * a.T + t) * a.Hq + hkv * a.G + g) * D + ch] = float_to_half_bits(r);
}

// ---- commit of accepted drafts ---------------------------------------------------------------------------------------------------------
// accepted[b]: indices of drafts, in order, up to the first one that is not in [0, T).  They are appended as decode steps would:
// rest rows, a flush of 64 tokens into the planes when the rest buffer fills (at most one: 63 + 64 < 128), column maxima, lengths.
constexpr int kCommitLayers = 16;      // layers per launch: their descriptors travel as kernel arguments
struct CommitArgs {
    akv_cache_layer c[kCommitLayers];
    const uint8_t *k[kCommitLayers], *v[kCommitLayers];
    const int *accepted;
    int T, A;
};

// grid (D / 16 * 2, B * Hkv, layers), 256 threads: a workgroup owns 16 channels of the keys (even blockIdx.x) or the values (odd) of one KV head.
__global__ __launch_bounds__(256) void tree_commit_kernel(CommitArgs a) {
    const akv_cache_layer &c = a.c[blockIdx.z];
    __shared__ unsigned short tile[2 * kRest][16 + 2];
    __shared__ int path[64];
    __shared__ int count_s;
    const bool is_v = blockIdx.x & 1;
    const int ch0 = (blockIdx.x >> 1) * 16, D = c.head_dim, H = c.n_kv_heads;
    const int b = blockIdx.y / H, h = blockIdx.y - b * H;
    const int n = max(0, c.seq_lens[b]), n_rest = n % kRest, flushed = n - n_rest;
    if (threadIdx.x < 64) {
        const int x = (int)threadIdx.x < a.A ? a.accepted[b * a.A + threadIdx.x] : -1;
        path[threadIdx.x] = x;
        const unsigned long long ok = __ballot(x >= 0 && x < a.T);
        // no further than the cache's capacity
        if (threadIdx.x == 0) count_s = max(0, min(ok == ~0ull ? 64 : (int)__builtin_ctzll(~ok), c.max_seq_len - n));
    }
    __syncthreads();
    const int count = count_s;
    if (count == 0) return;
    unsigned short *rest = reinterpret_cast<unsigned short *>(is_v ? c.restv : c.restk) + ((int64_t)b * kRest * H + h) * D + ch0;
    const unsigned short *draft = reinterpret_cast<const unsigned short *>(is_v ? a.v[blockIdx.z] : a.k[blockIdx.z]) + ((int64_t)b * a.T * H + h) * D + ch0;
    const int64_t row = (int64_t)H * D;
    const int total = n_rest + count;
    const bool flush = total >= kRest;
    // rows of the grown rest buffer: old ones only where they are flushed
    for (int id = threadIdx.x; id < total * 16; id += 256) {
        const int r = id >> 4, d = id & 15;
        if (r >= n_rest) tile[r][d] = draft[path[r - n_rest] * row + d];
        else if (flush) tile[r][d] = rest[r * row + d];
    }
    __syncthreads();
    uint8_t *colmax = (is_v ? c.v_exp_column_max : c.k_exp_column_max) + ((int64_t)b * H + h) * D + ch0;
    if (threadIdx.x < 16) {
        int mx = colmax[threadIdx.x];
        for (int r = n_rest; r < total; ++r) mx = max(mx, (tile[r][threadIdx.x] >> 10) & 31);
        colmax[threadIdx.x] = (uint8_t)mx;
    }
    if (!flush) {
        for (int id = threadIdx.x + n_rest * 16; id < total * 16; id += 256) rest[(id >> 4) * row + (id & 15)] = tile[id >> 4][id & 15];
        return;
    }
    for (int id = threadIdx.x + kRest * 16; id < total * 16; id += 256) rest[((id >> 4) - kRest) * row + (id & 15)] = tile[id >> 4][id & 15];
    const int64_t bh = (int64_t)b * H + h;
    if (is_v) {
        // token-major rows: 16 channels of a token are 16 + 8 + 8 bytes; a thread writes 4 channels
        const int r = threadIdx.x >> 2, d = (threadIdx.x & 3) * 4;
        const u32 w0 = tile[r][d], w1 = tile[r][d + 1], w2 = tile[r][d + 2], w3 = tile[r][d + 3];
        const int64_t at = (bh * c.max_seq_len + flushed + r) * D + ch0 + d;
        *reinterpret_cast<u32 *>(c.v_first_8 + at) = (w0 >> 8) | (w1 & 0xFF00u) | (w2 & 0xFF00u) << 8 | (w3 & 0xFF00u) << 16;
        *reinterpret_cast<unsigned short *>(c.v_mid_4 + at / 2) = (unsigned short)((w0 & 0xF0) | ((w1 >> 4) & 15) | (w2 & 0xF0) << 8 | ((w3 >> 4) & 15) << 8);
        *reinterpret_cast<unsigned short *>(c.v_last_4 + at / 2) = (unsigned short)((w0 & 15) << 4 | (w1 & 15) | (w2 & 15) << 12 | (w3 & 15) << 8);
    } else {
        // channel-major rows: 64 tokens of a channel are 64 + 32 + 32 bytes; a thread writes 4 tokens
        const int d = threadIdx.x >> 4, r = (threadIdx.x & 15) * 4;
        const u32 w0 = tile[r][d], w1 = tile[r + 1][d], w2 = tile[r + 2][d], w3 = tile[r + 3][d];
        const int64_t at = ((bh * c.n_max_blocks + flushed / c.k_block) * D + ch0 + d) * c.k_block + flushed % c.k_block + r;
        *reinterpret_cast<u32 *>(c.k_first_8 + at) = (w0 >> 8) | (w1 & 0xFF00u) | (w2 & 0xFF00u) << 8 | (w3 & 0xFF00u) << 16;
        *reinterpret_cast<unsigned short *>(c.k_mid_4 + at / 2) = (unsigned short)((w0 & 0xF0) | ((w1 >> 4) & 15) | (w2 & 0xF0) << 8 | ((w3 >> 4) & 15) << 8);
        *reinterpret_cast<unsigned short *>(c.k_last_4 + at / 2) = (unsigned short)((w0 & 15) << 4 | (w1 & 15) | (w2 & 15) << 12 | (w3 & 15) << 8);
    }
}

// The lengths, once every workgroup of the launch before has read them.
__global__ __launch_bounds__(64) void tree_commit_lens_kernel(CommitArgs a) {
    const akv_cache_layer &c = a.c[blockIdx.y];
    const int b = blockIdx.x;
    const int x = (int)threadIdx.x < a.A ? a.accepted[b * a.A + threadIdx.x] : -1;
    const unsigned long long ok = __ballot(x >= 0 && x < a.T);
    if (threadIdx.x == 0) {
        const int n = max(0, c.seq_lens[b]);
        c.seq_lens[b] = n + max(0, min(ok == ~0ull ? 64 : (int)__builtin_ctzll(~ok), c.max_seq_len - n));
    }
}

int check_layer(const akv_cache_layer *c, const char *what) {
    AKV_REQUIRE(c != nullptr, "%s: null descriptor", what);
    AKV_REQUIRE(c->k_first_8 && c->k_mid_4 && c->k_last_4 && c->v_first_8 && c->v_mid_4 && c->v_last_4 && c->k_exp_column_max &&
                    c->v_exp_column_max && c->restk && c->restv && c->seq_lens, "%s: null pointer in the layer", what);
    AKV_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "%s: head_dim %d: 64, 128 or 256", what, c->head_dim);
    AKV_REQUIRE(c->k_block == 64 || c->k_block == 256, "%s: k_block %d: 64 or 256", what, c->k_block);
    AKV_REQUIRE(c->bsz >= 1 && c->bsz <= 65535 && c->n_kv_heads >= 1 && (int64_t)c->bsz * c->n_kv_heads <= 65535,
                "%s: bsz %d x %d KV heads: at least 1 and at most 65535 together", what, c->bsz, c->n_kv_heads);
    AKV_REQUIRE(c->max_seq_len >= 1 && c->max_seq_len <= (1 << 30) && (int64_t)c->n_max_blocks * c->k_block >= c->max_seq_len / kRest * kRest,
                "%s: %d blocks of %d tokens for a capacity of %d", what, c->n_max_blocks, c->k_block, c->max_seq_len);
    const uintptr_t planes = (uintptr_t)c->k_first_8 | (uintptr_t)c->k_mid_4 | (uintptr_t)c->k_last_4 | (uintptr_t)c->v_first_8 |
                             (uintptr_t)c->v_mid_4 | (uintptr_t)c->v_last_4 | (uintptr_t)c->restk | (uintptr_t)c->restv;
    AKV_REQUIRE((planes & 15) == 0, "%s: planes and rest buffers must be 16-byte aligned", what);
    return AKV_OK;
}

// How a call is cut up: the rows of a KV head into groups of 16 or 32 (one or two matrix columns a lane), the planes into splits
// of whole tiles.
struct TreePlan {
    int nt, tok, groups, plane_splits, tiles_per_split, splits;
};
static TreePlan tree_plan(int bsz, int n_kv_heads, int rows, int bound) {
    TreePlan p;
    p.nt = rows > 16 ? 2 : 1;
    p.tok = p.nt == 2 ? 128 : 256;
    p.groups = (rows + 16 * p.nt - 1) / (16 * p.nt);
    const int flushed = bound / kRest * kRest, tiles = (flushed + p.tok - 1) / p.tok;
    const int64_t units = (int64_t)bsz * n_kv_heads * p.groups;
    int64_t want = (512 + units - 1) / units;                 // two workgroups per compute unit
    const int64_t most = (tiles + 3) / 4;                     // four waves take a tile each
    if (want > most) want = most;
    if (want < 1) want = 1;
    p.tiles_per_split = tiles > 0 ? (int)((tiles + want - 1) / want) : 1;
    p.plane_splits = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
    p.splits = p.plane_splits + 1;
    return p;
}

template <int D, int KB>
static void launch_tree(const TreeArgs &a, const TreePlan &p, bool cap, hipStream_t st) {
    const dim3 grid(p.splits, a.c.n_kv_heads * p.groups, a.c.bsz);
    const bool alibi = a.slopes != nullptr;
#define AKV_TREE(TPL, NT, CAP, ALIBI) hipLaunchKernelGGL((tree_kernel<D, KB, TPL, NT, CAP, ALIBI>), grid, dim3(256), 0, st, a)
#define AKV_TREE_NT(TPL, NT)                                                                                          \
    do {                                                                                                              \
        if (cap) { if (alibi) AKV_TREE(TPL, NT, true, true); else AKV_TREE(TPL, NT, true, false); }                   \
        else { if (alibi) AKV_TREE(TPL, NT, false, true); else AKV_TREE(TPL, NT, false, false); }                     \
    } while (0)
    if (p.nt == 2) AKV_TREE_NT(8, 2);
    else AKV_TREE_NT(16, 1);
#undef AKV_TREE_NT
#undef AKV_TREE
    hipLaunchKernelGGL(tree_combine_kernel<D>, dim3(a.rows, a.c.n_kv_heads, a.c.bsz), dim3(D), 0, st, a);
}

}  // namespace akv

extern "C" size_t akv_tree_attention_workspace_bytes(int bsz, int n_q_heads, int n_kv_heads, int head_dim, int n_drafts, int len_bound) {
    if (bsz < 1 || n_q_heads < 1 || n_kv_heads < 1 || n_q_heads % n_kv_heads || head_dim < 1 || n_drafts < 1 || n_drafts > 64 || len_bound < 0) return 0;
    const int rows = n_q_heads / n_kv_heads * n_drafts;
    const akv::TreePlan p = akv::tree_plan(bsz, n_kv_heads, rows, len_bound);
    return (size_t)bsz * n_kv_heads * p.splits * rows * (head_dim + 2) * sizeof(float);
}

extern "C" int akv_tree_attention(const akv_cache_layer *layer, const uint8_t *q, const uint8_t *k, const uint8_t *v, const int64_t *ancestors,
                                  int ancestors_per_sequence, const float *slopes, float scale, float softcap, uint8_t *out, int n_drafts,
                                  int n_q_heads, int len_bound, void *workspace, size_t workspace_bytes, akv_stream_t stream) {
    const int rc = akv::check_layer(layer, "tree_attention");
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(q && k && v && ancestors && out, "tree_attention: null pointer");
    AKV_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0, "tree_attention: q, k, v and out must be 16-byte aligned");
    AKV_REQUIRE(n_drafts >= 1 && n_drafts <= 64, "tree_attention: %d drafts: 1 to 64", n_drafts);
    AKV_REQUIRE(n_q_heads >= 1 && n_q_heads % layer->n_kv_heads == 0, "tree_attention: heads %d / %d", n_q_heads, layer->n_kv_heads);
    AKV_REQUIRE(len_bound >= 0 && len_bound <= layer->max_seq_len, "tree_attention: len_bound %d outside [0, %d]", len_bound, layer->max_seq_len);
    AKV_REQUIRE(scale > 0.f && scale < 1e30f, "tree_attention: scale %g must be positive and finite", scale);
    AKV_REQUIRE(softcap >= 0.f && softcap < 1e30f, "tree_attention: softcap %g must be zero (off) or positive and finite", softcap);
    const size_t need = akv_tree_attention_workspace_bytes(layer->bsz, n_q_heads, layer->n_kv_heads, layer->head_dim, n_drafts, len_bound);
    AKV_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0, "tree_attention: needs a 16-byte aligned workspace of %zu bytes, got %zu",
                need, workspace_bytes);
    akv::TreeArgs a;
    a.c = *layer;
    a.q = q; a.k = k; a.v = v;
    a.anc = reinterpret_cast<const unsigned long long *>(ancestors);
    a.anc_stride = ancestors_per_sequence ? n_drafts : 0;
    a.slopes = slopes;
    a.out = out;
    a.parts = static_cast<float *>(workspace);
    a.T = n_drafts; a.Hq = n_q_heads; a.G = n_q_heads / layer->n_kv_heads; a.rows = a.T * a.G;
    a.form = akv::score_form(scale, softcap);
    const akv::TreePlan p = akv::tree_plan(layer->bsz, layer->n_kv_heads, a.rows, len_bound);
    a.plane_splits = p.plane_splits; a.tiles_per_split = p.tiles_per_split; a.splits = p.splits;
    AKV_REQUIRE((int64_t)layer->n_kv_heads * p.groups <= 65535, "tree_attention: too many rows");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool cap = softcap > 0.f;
    if (layer->k_block == 64) {
        if (layer->head_dim == 64) akv::launch_tree<64, 64>(a, p, cap, st);
        else if (layer->head_dim == 128) akv::launch_tree<128, 64>(a, p, cap, st);
        else akv::launch_tree<256, 64>(a, p, cap, st);
    } else {
        if (layer->head_dim == 64) akv::launch_tree<64, 256>(a, p, cap, st);
        else if (layer->head_dim == 128) akv::launch_tree<128, 256>(a, p, cap, st);
        else akv::launch_tree<256, 256>(a, p, cap, st);
    }
    return akv::check_launch("tree_attention");
}

extern "C" int akv_tree_commit(const akv_cache_layer *layers, int n_layers, const uint8_t *const *k, const uint8_t *const *v, const int *accepted,
                               int n_drafts, int n_accepted, akv_stream_t stream) {
    AKV_REQUIRE(layers && k && v && accepted, "tree_commit: null pointer");
    AKV_REQUIRE(n_layers >= 1, "tree_commit: %d layers", n_layers);
    AKV_REQUIRE(n_drafts >= 1 && n_drafts <= 64, "tree_commit: %d drafts: 1 to 64", n_drafts);
    AKV_REQUIRE(n_accepted >= 1 && n_accepted <= 64, "tree_commit: %d accepted drafts: 1 to 64", n_accepted);
    for (int i = 0; i < n_layers; ++i) {
        const int rc = akv::check_layer(layers + i, "tree_commit");
        if (rc != AKV_OK) return rc;
        AKV_REQUIRE(k[i] && v[i], "tree_commit: null pointer");
        AKV_REQUIRE(layers[i].bsz == layers[0].bsz && layers[i].n_kv_heads == layers[0].n_kv_heads && layers[i].head_dim == layers[0].head_dim,
                    "tree_commit: layer %d has another shape than layer 0", i);
        for (int j = 0; j < i; ++j)
            AKV_REQUIRE(layers[i].seq_lens != layers[j].seq_lens, "tree_commit: layers %d and %d share their lengths", j, i);
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    for (int first = 0; first < n_layers; first += akv::kCommitLayers) {
        const int count = n_layers - first < akv::kCommitLayers ? n_layers - first : akv::kCommitLayers;
        akv::CommitArgs a;
        for (int i = 0; i < count; ++i) {
            a.c[i] = layers[first + i];
            a.k[i] = k[first + i];
            a.v[i] = v[first + i];
        }
        a.accepted = accepted;
        a.T = n_drafts;
        a.A = n_accepted;
        hipLaunchKernelGGL(akv::tree_commit_kernel, dim3(layers[0].head_dim / 16 * 2, layers[0].bsz * layers[0].n_kv_heads, count), dim3(256), 0, st, a);
        hipLaunchKernelGGL(akv::tree_commit_lens_kernel, dim3(layers[0].bsz, count), dim3(64), 0, st, a);
    }
    return akv::check_launch("tree_commit");
}
