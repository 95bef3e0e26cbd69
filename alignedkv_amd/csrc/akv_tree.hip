// Attention of a tree of drafted tokens over the split-plane cache, and the commit of the drafts that were accepted.
//
// T drafted tokens per sequence attend to the whole cache (planes and rest buffer, every plane: a row of planes is needed
// at full precision as soon as one of the T x G query rows of a KV head needs it) and to the drafts in their ancestors'
// bit mask.  The cache does not change until tree_commit appends the accepted path.
#include "akv_attention.h"

namespace akv {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
constexpr int kRest = 64;       // tokens of the rest buffer

struct TreeArgs {
    akv_cache_layer c;
    const uint8_t *q, *k, *v;             // fp16 [B, T, Hq | Hkv, D]
    const unsigned long long *anc;        // [T] or [B, T]
    int anc_stride;                       // T or 0
    const float *slopes;
    uint8_t *out;
    float *parts;                         // [Hkv, splits, rows] x {D sums}, then the same x {m, l}
    int *shares;                          // [B] x {first split, splits}
    int T, Hq, G, rows;                   // rows = T * G
    int log_tokens, splits, own_tail;     // of a round's tokens; of all sequences together, for a KV head; the tail has a split of its own
    ScoreForm form;
};

// Cached tokens of a sequence, kept inside the planes whatever the device holds.
__device__ __forceinline__ int cached_tokens(const TreeArgs &a, int b) { return max(0, min(a.c.seq_lens[b], a.c.max_seq_len)); }

// Which stretch of which sequence split u is.  The splits are dealt out by the lengths: every one takes the same number of rounds, the
// fewest with which all sequences together need no more than there are, so that a ragged batch does not wait for its longest sequence (8
// sequences of 1000 to 8000 tokens, 8 KV heads x 128, 5 drafts: 47 us against 59 with as many splits for each, 32 of 100 to 9400 131 against 156).
struct Share {
    int b, split, count, tokens;      // tokens: of a split of the planes
};
// Rounds of a split: an odd number where it is not small, so that splits that run side by side do not start a power of two apart in memory,
// which crowds them on the same memory channels (8 x 4096 tokens x 32 heads: 116 -> 112 us).
__device__ __forceinline__ int odd_rounds(int per) { return per >= 8 ? per | 1 : per; }
// ceil(a / b) for 0 <= a <= 2^24, 0 < b (more rounds than that do not fit the memory; the quotient before it is cut off is then wrong by
// less than one: 2^-23 and 2^-24 of at most 2^24 / 3, and exact for one and two; an integer division is three times as long, and a workgroup waits for this)
__device__ __forceinline__ int ceil_div(int a, int b) {
    int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));       // off by one at most
    int rest = a - q * b;
    if (rest < 0) rest += b, --q;
    return q + (rest > 0 ? 1 : 0) + (rest > b ? 1 : 0);
}
__device__ __forceinline__ bool find_share(const TreeArgs &a, int u, Share &s) {
    const int B = a.c.bsz, lane = threadIdx.x & 63, least = 1 - a.own_tail, planes = a.splits - B * a.own_tail;
    const auto rounds_of = [&](int b) { return (cached_tokens(a, b) / kRest * kRest + (1 << a.log_tokens) - 1) >> a.log_tokens; };
    if (B == 1) {
        const int r = rounds_of(0), per = odd_rounds(max(1, ceil_div(r, planes)));
        s = {0, u, max(least, ceil_div(r, per)) + a.own_tail, per << a.log_tokens};
        return u < s.count;
    }
    if (planes == B && !a.own_tail) {           // one each, whatever the lengths (more than 512 sequences: always)
        s = {u, 0, 1, 1 << 30};
        return u < B;
    }
    // a lane a sequence, 64 at a time; -1: none.  (Those beyond the first 64 are read again in every loop: in registers, the loops unrolled, 300
    // sequences take 82 us instead of 86, but 4 with head_dim 256 89 instead of 84.)
    const int r0 = lane < B ? rounds_of(lane) : -1;
    const auto rounds_at = [&](int c) { return c == 0 ? r0 : (c + lane < B ? rounds_of(c + lane) : -1); };
    const auto splits_of = [&](int r, int per) { return r < 0 ? 0 : max(least, ceil_div(r, per)) + a.own_tail; };
    int all = 0, longest = 1;
    for (int c = 0; c < B; c += 64) {
        const int r = rounds_at(c);
        all += wave_sum_i32(max(r, 0));
        longest = max(longest, (int)~wave_min_u32(~(u32)max(r, 0)));
    }
    int lo = max(1, (int)((u32)(all + planes - 1) / (u32)planes)), hi = longest;
    const int spare = planes - B;       // (a sequence needs fewer than r / per + 1 splits of its planes)
    if (spare > 0) hi = min(hi, max(lo, (int)((u32)(all + spare - 1) / (u32)spare)));
    int per = lo;
    while (lo < hi) {
        int need = 0;
        for (int c = 0; c < B; c += 64) need += wave_sum_i32(splits_of(rounds_at(c), per));
        if (need <= a.splits) hi = per;
        else lo = per + 1;
        per = (lo + hi) >> 1;
    }
    per = odd_rounds(hi);
    int before = 0;
    for (int c = 0; c < B; c += 64) {
        const int n = splits_of(rounds_at(c), per);
        int inc = n;
        const int in_chunk = min(B - c, 64);
        for (int d = 1; d < in_chunk; d <<= 1) {
            const int o = __shfl_up(inc, d);
            if (lane >= d) inc += o;
        }
        const unsigned long long past = __ballot(u < before + inc);
        if (past) {
            const int l = __builtin_ctzll(past), count = __builtin_amdgcn_readlane(n, l);
            s = {c + l, u - (before + __builtin_amdgcn_readlane(inc, l) - count), count, per << a.log_tokens};
            return true;
        }
        before += __builtin_amdgcn_readlane(inc, in_chunk - 1);
    }
    return false;
}

// 16-bit values of elements 0,2 / 1,3 / 4,6 / 5,7 of 8 elements (high bytes Ha, Hb; nibbles M, L).  They are used in this order: four
// elements 0 1 2 3 lie at places 0 2 1 3, which costs nothing where the order of tokens or channels is free.
__device__ __forceinline__ u32x4 rebuild8(u32 Ha, u32 Hb, u32 M, u32 L) {
    u32 E, O;
    split_even_odd(M, L, E, O);
    return u32x4{__builtin_amdgcn_perm(Ha, E, 0x06010400u), __builtin_amdgcn_perm(Ha, O, 0x07010500u), __builtin_amdgcn_perm(Hb, E, 0x06030402u),
                 __builtin_amdgcn_perm(Hb, O, 0x07030502u)};
}
__host__ __device__ constexpr int place(int x) { return (x & ~3) | (x & 1) << 1 | (x >> 1 & 1); }    // (its own inverse)
// eight fp16 values in memory order, brought into that order
__device__ __forceinline__ u32x4 placed(u32x4 w) {
    return u32x4{__builtin_amdgcn_perm(w.y, w.x, 0x05040100u), __builtin_amdgcn_perm(w.y, w.x, 0x07060302u), __builtin_amdgcn_perm(w.w, w.z, 0x05040100u),
                 __builtin_amdgcn_perm(w.w, w.z, 0x07060302u)};
}

// 16 elements of a plane triple: one channel of 16 tokens (keys) or 16 channels of one token (values).
struct Raw16 {
    u32x4 h;
    u32x2 m, l;
};
// (off: of the high bytes; kSkip and a little beyond it are out of every range, halved too)
__device__ __forceinline__ Raw16 load_raw16(__amdgpu_buffer_rsrc_t rh, __amdgpu_buffer_rsrc_t rm, __amdgpu_buffer_rsrc_t rl, u32 off) {
    Raw16 r;
    r.h = __builtin_amdgcn_raw_buffer_load_b128(rh, (int)off, 0, 0);
    r.m = __builtin_amdgcn_raw_buffer_load_b64(rm, (int)(off >> 1), 0, 0);
    r.l = __builtin_amdgcn_raw_buffer_load_b64(rl, (int)(off >> 1), 0, 0);
    return r;
}

// Keys in LDS: [channel][BN tokens] fp16, as the planes have them.  The operand of a score product wants eight channels of one
// token a lane: two transposing reads of four channels each.
template <int BN>
__device__ __forceinline__ int key_byte(int channel, int chunk) {
    if constexpr (BN == 64) return tile_byte<64>(channel, chunk);
    return channel * 64 + chunk * 16;      // (a read takes whole rows here: they do not collide)
}
template <int D, int BN>
__device__ __forceinline__ void key_scores(f32x16 (&acc)[BN / 32], const uint8_t *k_tile, int at0, int at1, const f16x8 (&qf)[D / 16]) {
#pragma unroll
    for (int tb = 0; tb < BN / 32; ++tb)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[tb][r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int tb = 0; tb < BN / 32; ++tb) {
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(k_tile + (at0 ^ (tb << 6)) + ks * 16 * BN * 2));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(k_tile + (at1 ^ (tb << 6)) + ks * 16 * BN * 2));
            acc[tb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)), qf[ks], acc[tb], 0, 0, 0);
        }
        if (ks % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
}

// o_t = sum_j softmax_j(cap(scale q_t . k_j) - slope (pos_t - pos_j)) v_j over the cache and the drafts that t sees, one pass with a running
// maximum and sum in 32 bits; probabilities go to fp16 for the second product (2^-11 of each, or 2^-32 of the split's
// largest; its sums are in 32 bits).
// Bound by the planes' bytes while a KV head has few rows (one draft, 8 x 4096 tokens x 32 heads x 128: 102 to 106 us with the join, 5.1 to 5.3 TB/s), by what the
// vector units do for a score beside the products -- unpacking, scaling, one exponential -- where it has many (64 drafts x 4 heads a KV head over
// 4 x 32768, biased: 203 us, 677 TFLOP/s).
// grid: a workgroup per split, row group and KV head (see unit below).  A sequence's splits: stretches of the planes; the last one: the rest buffer and the
// drafts, behind its stretch unless the tail has a split of its own.  A round takes TT = PARTS * BN tokens: their planes are loaded into registers while the round before is computed,
// unpacked once (one instruction an element) and put into LDS as fp16, and each wave multiplies 32 query rows with BN of them:
// THREADS / 2 / PARTS rows a workgroup, so few rows do not leave waves idle.  The parts' sums are joined through LDS, the splits' by
// tree_combine_kernel.
template <int D, int KB, int PARTS, int BN, int THREADS, bool CAP, bool ALIBI>
__global__ __launch_bounds__(THREADS, D == 256 ? 1 : 2) void tree_kernel(TreeArgs a) {
    constexpr int TT = PARTS * BN, ROWS = THREADS / 2 / PARTS, WAVES = THREADS / 64 / PARTS, TB = BN / 32;
    constexpr int UNITS = D * TT / 16 / THREADS;         // Raw16 of each side per thread and round
    constexpr int kPart = D * BN * 2;
    constexpr int kBox = 64 * (D / 2 + 2 + D / 32);  // words a wave hands over when the parts are joined
    constexpr int kBuffers = PARTS == 1 ? 2 : 1, kBuffer = 2 * PARTS * kPart;
    constexpr int kLds = kBuffers * kBuffer > (PARTS - 1) * WAVES * kBox * 4 ? kBuffers * kBuffer : (PARTS - 1) * WAVES * kBox * 4;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
    __shared__ int tail_pos[128];                    // positions of the tail's tokens
    __shared__ int odd_tile[PARTS];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_index(), half = lane >> 5, part = wave / WAVES, part_tid = tid & (64 * WAVES - 1);
    const int groups = (a.rows + ROWS - 1) / ROWS;
    // Workgroups are dealt out to the 8 XCDs in turn: the row groups of a stretch of the planes are 8 apart, so that one XCD's L2 serves
    // them all.
    const int unit = (int)(blockIdx.x / 8 / groups) * 8 + (int)(blockIdx.x % 8), rg = blockIdx.x / 8 % groups;
    const int hkv = unit / a.splits, slot = unit - hkv * a.splits;
    Share share;
    if (hkv >= a.c.n_kv_heads || !find_share(a, slot, share)) return;
    const int b = share.b, split = share.split;
    if (hkv == 0 && rg == 0 && split == 0 && tid == 0) *reinterpret_cast<i32x2 *>(a.shares + 2 * b) = i32x2{slot, share.count};
    const int n = cached_tokens(a, b), flushed = n / kRest * kRest, n_rest = n - flushed, total = n_rest + a.T;
    const int64_t bh = (int64_t)b * a.c.n_kv_heads + hkv;
    const int row = rg * ROWS + (wave % WAVES) * 32 + (lane & 31), row_c = min(row, a.rows - 1), g = row_c / a.T, t = row_c - g * a.T;
    const bool tail = split == share.count - 1;
    uint8_t *kt = lds + part * kPart, *vt = lds + PARTS * kPart + part * kPart;

    // the planes: this thread's pieces of a round
    const int first = split * share.tokens, end = split < share.count - a.own_tail ? min(first + share.tokens, flushed) : 0;
    Raw16 kr[UNITS], vr[UNITS];
    // Piece u of a thread lies a constant behind piece 0, in memory and in LDS: four addresses stay in registers.
    constexpr int kChStep = THREADS * 16 / TT, kTokStep = THREADS * 16 / D;      // channels / tokens from piece to piece
    static_assert(kChStep % 16 == 0 && kTokStep % 16 == 0, "rows 16 apart are laid out alike");
    const int k_tok = tid % (TT / 16) * 16, k_ch = tid / (TT / 16), v_c16 = tid % (D / 16), v_tok = tid / (D / 16);
    int k_lds = k_tok / BN * kPart + key_byte<BN>(k_ch, k_tok % BN / 8);                                // the other half: ^ 16
    int v_lds = PARTS * kPart + v_tok / BN * kPart + tile_byte<D>(place(v_tok % BN), 2 * v_c16);
    int v_off = v_tok * D + v_c16 * 16;
    auto request_k = [&](int j0) {
        const int64_t blk = bh * a.c.n_max_blocks + j0 / KB;
        const int blocks = min(KB == 64 && TT > 64 ? TT / 64 : 1, a.c.n_max_blocks - j0 / KB);
        const auto rh = make_rsrc(a.c.k_first_8 + blk * (D * KB), blocks * D * KB);
        const auto rm = make_rsrc(a.c.k_mid_4 + blk * (D * KB / 2), blocks * D * KB / 2);
        const auto rl = make_rsrc(a.c.k_last_4 + blk * (D * KB / 2), blocks * D * KB / 2);
        const int in = j0 % KB + k_tok;
        const u32 off = j0 + k_tok < end ? in / KB * (D * KB) + k_ch * KB + in % KB : kSkip;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) kr[u] = load_raw16(rh, rm, rl, off + u * (kChStep * KB));
    };
    auto request_v = [&](int j0) {
        const int64_t r0 = bh * a.c.max_seq_len + j0;
        const int rows = min(end - j0, TT);                   // (rows behind them are out of range)
        const auto rh = make_rsrc(a.c.v_first_8 + r0 * D, rows * D);
        const auto rm = make_rsrc(a.c.v_mid_4 + r0 * (D / 2), rows * D / 2);
        const auto rl = make_rsrc(a.c.v_last_4 + r0 * (D / 2), rows * D / 2);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) vr[u] = load_raw16(rh, rm, rl, v_off + u * (kTokStep * D));
    };
    auto put = [&](int at, int step, const Raw16 (&raw)[UNITS]) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            *reinterpret_cast<u32x4 *>(lds + at + u * step) = rebuild8(raw[u].h.x, raw[u].h.y, raw[u].m.x, raw[u].l.x);
            *reinterpret_cast<u32x4 *>(lds + (at ^ 16) + u * step) = rebuild8(raw[u].h.z, raw[u].h.w, raw[u].m.y, raw[u].l.y);
        }
    };
    // (V of a round is asked for behind its K: both at once do not fit beside the sums, except where a wave has a SIMD to itself)
    constexpr bool kAhead = !(D == 256 && PARTS == 4);
    if (first < end) {
        request_k(first);
        if constexpr (kAhead) request_v(first);
    }

    f16x8 qf[D / 16];
    const uint8_t *qp = a.q + (((int64_t)b * a.T + t) * a.Hq + hkv * a.G + g) * (D * 2);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *reinterpret_cast<const f16x8 *>(qp + (2 * ks + half) * 16);
    const unsigned long long *anc = a.anc + (int64_t)b * a.anc_stride;
    const unsigned long long named = ~0ull >> (64 - a.T);       // bits at and beyond T name no draft
    const unsigned long long my_anc = anc[t] & named;
    const int pos = n + __popcll(my_anc & ~(1ull << t));
    const float neg_slope = ALIBI ? a.slopes[hkv * a.G + g] * -kLog2e : 0.f;
    LaneBytes<D> at;
    const int kr0 = 8 * half + ((lane & 15) >> 2), kchunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    int k_at0 = key_byte<BN>(kr0, kchunk) + (lane & 1) * 8, k_at1 = key_byte<BN>(kr0 + 4, kchunk) + (lane & 1) * 8;
    f32x16 o[D / 32];
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[cb][r] = 0.f;
    RowState st;
    OddValues<D> odd;

    if constexpr (kBuffers == 2) {
        // the next round's keys and values go into the other buffer while this one's are multiplied: one barrier a round (64 drafts x 4 heads
        // over 4 x 32768: 234 us against 257 with one buffer and two barriers; with more parts two buffers do not leave room for a second
        // workgroup)
        if (first < end) {
            put(k_lds, kChStep * BN * 2, kr);
            put(v_lds, kTokStep * D * 2, vr);
            if (first + TT < end) {
                request_k(first + TT);
                request_v(first + TT);
            }
        }
        lds_barrier();
        int buf = 0;
        for (int j0 = first; j0 < end; j0 += TT) {
            at.pin();
            asm volatile("" : "+v"(k_at0), "+v"(k_at1), "+v"(k_lds), "+v"(v_lds), "+v"(v_off));
            const int next = j0 + TT, other = buf ^ kBuffer;
            f32x16 x[TB];
            f16x8 p[TB][2];
            key_scores<D, BN>(x, kt + buf, k_at0, k_at1, qf);
            if (next < end) {
                put(k_lds + other, kChStep * BN * 2, kr);
                if (next + TT < end) request_k(next + TT);
            }
            const float factor = modify_block<CAP, TB>(x, a.form);
            float shift = 0.f;
            if constexpr (ALIBI) {
                // every cached token lies before the row: the distance is linear in the token
                const float s = neg_slope * __builtin_amdgcn_rcpf(factor);       // (the same in every lane; times factor again: 1 ulp of the bias)
                shift = -neg_slope * (float)(j0 + 4 * half - pos);
#pragma unroll
                for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[tb][r] = fmaf(-s, (float)(tb * 32 + 8 * (r >> 2) + place(r & 3)), x[tb][r]);
            }
            tile_softmax<D, BN>(x, factor, shift, st, o, p);
            if (next < end) {
                put(v_lds + other, kTokStep * D * 2, vr);
                if (next + TT < end) request_v(next + TT);
            }
            tile_output<D, BN>(o, vt + buf, at, p);
            lds_barrier();
            buf = other;
        }
    } else
    for (int j0 = first; j0 < end; j0 += TT) {
        at.pin();
        asm volatile("" : "+v"(k_at0), "+v"(k_at1), "+v"(k_lds), "+v"(v_lds), "+v"(v_off));
        put(k_lds, kChStep * BN * 2, kr);
        const int next = j0 + TT;
        if constexpr (kAhead) {
            if (next < end) request_k(next);
        } else {
            request_v(j0);
        }
        lds_barrier();
        const int jp = j0 + part * BN;              // this wave's tokens: whole 64s or none (32: the valid ones come first)
        const bool mine = jp < end;
        f32x16 x[TB];
        f16x8 p[TB][2];
        float factor = 1.f, shift = 0.f;
        if (mine) {
            key_scores<D, BN>(x, kt, k_at0, k_at1, qf);
            factor = modify_block<CAP, TB>(x, a.form);
            if constexpr (ALIBI) {
                // every cached token lies before the row: the distance is linear in the token
                const float s = neg_slope * __builtin_amdgcn_rcpf(factor);       // (the same in every lane; times factor again: 1 ulp of the bias)
                shift = -neg_slope * (float)(jp + 4 * half - pos);
#pragma unroll
                for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[tb][r] = fmaf(-s, (float)(tb * 32 + 8 * (r >> 2) + place(r & 3)), x[tb][r]);
            }
            tile_softmax<D, BN>(x, factor, shift, st, o, p);
        }
        put(v_lds, kTokStep * D * 2, vr);
        if (next < end) {
            if constexpr (kAhead) request_v(next);
            else request_k(next);
        }
        lds_barrier();
        if (mine) tile_output<D, BN>(o, vt, at, p);
    }

    if (tail) {
        // the rest buffer and the drafts: fp16 rows, keys and values token-major in LDS
        const int H = a.c.n_kv_heads;
        const int64_t row_bytes = (int64_t)H * D * 2, r0 = ((int64_t)b * kRest * H + hkv) * (D * 2), d0 = ((int64_t)b * a.T * H + hkv) * (D * 2);
        if (tid < total) tail_pos[tid] = tid < n_rest ? flushed + tid : n + __popcll(anc[tid - n_rest] & named & ~(1ull << (tid - n_rest)));
        if (tid < PARTS) odd_tile[tid] = -1;
        constexpr int CPR = D / 8;
        for (int u0 = 0; u0 < total; u0 += TT) {
            lds_barrier();
#pragma unroll 2
            for (int id = tid; id < TT * CPR; id += THREADS) {
                const int u = id / CPR, ch = id % CPR, uu = u0 + u;
                u32x4 kw = {0u, 0u, 0u, 0u}, vw = {0u, 0u, 0u, 0u};
                if (uu < total) {
                    const bool old = uu < n_rest;
                    const int64_t off = (old ? r0 + uu * row_bytes : d0 + (uu - n_rest) * row_bytes) + ch * 16;
                    kw = *reinterpret_cast<const u32x4 *>((old ? a.c.restk : a.k) + off);
                    vw = *reinterpret_cast<const u32x4 *>((old ? a.c.restv : a.v) + off);
                }
                *reinterpret_cast<u32x4 *>(lds + u / BN * kPart + tile_byte<D>(u % BN, ch)) = kw;
                *reinterpret_cast<u32x4 *>(lds + PARTS * kPart + u / BN * kPart + tile_byte<D>(u % BN, ch)) = placed(vw);
            }
            lds_barrier();
            const int up = u0 + part * BN;
            const auto token = [&](int c) { return up + 4 * half + (c >> 4) * 32 + 8 * ((c & 15) >> 2) + (c & 3); };   // of register c % 16 of block c / 16
            u32 seen = 0;
#pragma unroll
            for (int c = 0; c < TB * 16; ++c) {
                const int u = token(c);
                seen |= u < n_rest || (u < total && ((my_anc >> ((u - n_rest) & 63)) & 1)) ? 1u << c : 0u;
            }
            if (up < total && share_nonfinite<D, BN, 64 * WAVES>(vt, part_tid)) odd_tile[part] = u0;
            lds_barrier();
            bool found = false;
#pragma unroll
            for (int s = 0; s < PARTS; ++s) found = found || odd_tile[s] == u0;
            if (found) {
                note_nonfinite<D, BN>(odd, vt, at, seen);
                lds_barrier();
                zero_nonfinite_tile<D, BN, 64 * WAVES>(vt, part_tid);
                lds_barrier();
            }
            if (up < total) {
                f32x16 x[TB];
                f16x8 p[TB][2];
                tile_scores<D, BN>(x, kt, at, qf);
                const float factor = modify_block<CAP, TB>(x, a.form);
                const float s = ALIBI ? neg_slope / factor : 0.f;
#pragma unroll
                for (int c = 0; c < TB * 16; ++c) {
                    float y = x[c >> 4][c & 15];
                    if constexpr (ALIBI) y = fmaf(s, fabsf((float)(pos - tail_pos[min(token(c), total - 1)])), y);
                    x[c >> 4][c & 15] = (seen >> c) & 1 ? y : kNegInf;
                    if (c % 8 == 7) __builtin_amdgcn_sched_barrier(0);
                }
                tile_softmax<D, BN>(x, factor, 0.f, st, o, p);
                tile_output<D, BN>(o, vt, at, p);
            }
        }
    }

    float l = halves_sum(st.l);
    if (odd.any()) odd.add(o);
    if constexpr (PARTS > 1) {
        lds_barrier();
        float *box = reinterpret_cast<float *>(lds) + lane;
        if (part > 0) {
            float *to = box + ((part - 1) * WAVES + wave % WAVES) * kBox;
#pragma unroll
            for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
                for (int r = 0; r < 16; ++r) to[(cb * 16 + r) * 64] = o[cb][r];
            to[(D / 2) * 64] = st.m;
            to[(D / 2 + 1) * 64] = l;
        }
        lds_barrier();
        if (part > 0) return;
        float m = st.m;
#pragma unroll
        for (int s = 1; s < PARTS; ++s) m = fmaxf(m, box[((s - 1) * WAVES + wave) * kBox + (D / 2) * 64]);
        const float f0 = st.m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(st.m - m);
        l *= f0;
#pragma unroll
        for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[cb][r] *= f0;
#pragma unroll
        for (int s = 1; s < PARTS; ++s) {
            const float *from = box + ((s - 1) * WAVES + wave) * kBox;
            const float ms = from[(D / 2) * 64], f = ms == kNegInf ? 0.f : __builtin_amdgcn_exp2f(ms - m);
            l = fmaf(from[(D / 2 + 1) * 64], f, l);
#pragma unroll
            for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[cb][r] = fmaf(from[(cb * 16 + r) * 64], f, o[cb][r]);
        }
        st.m = m;
    }
    if (row >= a.rows) return;
    float *po = a.parts + ((int64_t)unit * a.rows + row) * D;
    float *pm = a.parts + (int64_t)a.c.n_kv_heads * a.splits * a.rows * D + ((int64_t)unit * a.rows + row) * 2;
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4 *>(po + cb * 32 + 8 * q + 4 * half) = f32x4{o[cb][4 * q], o[cb][4 * q + 2], o[cb][4 * q + 1], o[cb][4 * q + 3]};
    if (half == 0) {
        pm[0] = st.m;
        pm[1] = l;
    }
}

// Joins the splits of a row in order: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  D / 4 lanes a row, four channels a lane, four splits'
// sums requested at a time: latency and the sums' bytes (4 to 9 us behind a call's 14 to 203).  Joined in the order of the splits, so that the
// bits do not depend on which workgroup ends first.
template <int D>
__global__ __launch_bounds__(256) void tree_combine_kernel(TreeArgs a) {
    constexpr int LANES = D / 4, ROWS = 256 / LANES;
    const int row = blockIdx.x * ROWS + threadIdx.x / LANES, hkv = blockIdx.y, b = blockIdx.z, ch = threadIdx.x % LANES * 4;
    if (row >= a.rows) return;
    const i32x2 share = *reinterpret_cast<const i32x2 *>(a.shares + 2 * b);
    const int splits = share.y;
    const int64_t first = (int64_t)hkv * a.splits + share.x, step = (int64_t)a.rows * D;
    const float *po = a.parts + first * step + (int64_t)row * D + ch;
    const f32x2 *pm = reinterpret_cast<const f32x2 *>(a.parts + (int64_t)a.c.n_kv_heads * a.splits * step) + first * a.rows + row;
    float m = kNegInf, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += 4) {
        f32x4 x[4];
        f32x2 ml[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = min(s0 + i, splits - 1);
            x[i] = *reinterpret_cast<const f32x4 *>(po + s * step);
            ml[i] = pm[(int64_t)s * a.rows];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (s0 + i >= splits) break;
            const float top = fmaxf(m, ml[i].x);
            const float f0 = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m - top), f1 = ml[i].x == kNegInf ? 0.f : __builtin_amdgcn_exp2f(ml[i].x - top);
            o = o * f0 + x[i] * f1;
            l = l * f0 + ml[i].y * f1;
            m = top;
        }
    }
    const float r = l == 0.f ? 1.f : 1.f / l;      // (a row that saw nothing: zeros)
    const int g = row / a.T, t = row - g * a.T;
    *reinterpret_cast<u32x2 *>(a.out + ((((int64_t)b * a.T + t) * a.Hq + hkv * a.G + g) * D + ch) * 2) = u32x2{pack_f16(o[0] * r, o[1] * r), pack_f16(o[2] * r, o[3] * r)};
}

// ---- commit of accepted drafts ---------------------------------------------------------------------------------------------------------
// accepted[b]: indices of drafts, in order, up to the first one that is not in [0, T).  They are appended as decode steps would:
// rest rows, a flush of 64 tokens into the planes when the rest buffer fills (at most one: 63 + 64 < 128), column maxima, lengths.
// One layer is latency: lengths, then indices, then rows, each a round trip, and few bytes behind them (32 heads x 128: 3.6 us and 1.7 for the
// lengths).  All layers of a model go into one launch, their descriptors as kernel arguments (24 layers x 8 sequences x 8 heads x 128, 16 drafts: 15
// us where the caches' lines are in L2, 19 where not, and 2 to 4 for the lengths; a launch a layer: 79 us): 6144 workgroups of 17 KB LDS, of which eight share a
// compute unit, are three rounds of the chip, and each round waits for those round trips.
constexpr int kCommitLayers = 30;      // (4 KB of arguments)
struct CommitLayer {
    uint8_t *k_first_8, *k_mid_4, *k_last_4, *v_first_8, *v_mid_4, *v_last_4, *k_max, *v_max, *restk, *restv;
    const int *seq_lens;
    const uint8_t *k, *v;
    int n_max_blocks, max_seq_len, k_block;
};
struct CommitArgs {
    CommitLayer c[kCommitLayers];
    const int *accepted;
    int T, A, H;
};
static_assert(sizeof(CommitArgs) <= 4096, "kernel arguments");

// How many of `accepted` are appended to a cache of n tokens: up to the first index outside [0, T), no further than the capacity.
__device__ __forceinline__ int accepted_count(int index, int T, int n, int capacity) {
    const unsigned long long ok = __ballot(index >= 0 && index < T);
    return max(0, min(ok == ~0ull ? 64 : (int)__builtin_ctzll(~ok), capacity - n));
}

// grid (2 * D / 64, B * Hkv, layers), 256 threads: 64 channels of the keys (even blockIdx.x) or the values of one KV head: the tile
// then takes 17 KB of LDS and eight workgroups share a compute unit.
template <int D>
__global__ __launch_bounds__(256) void tree_commit_kernel(CommitArgs a) {
    const CommitLayer &c = a.c[blockIdx.z];
    constexpr int CH = 64, PITCH = CH + 2, LANES = CH / 4;          // a row of the tile in halves; threads to a row, four channels each
    __shared__ __attribute__((aligned(16))) unsigned short tile[2 * kRest * PITCH];
    const bool is_v = blockIdx.x & 1;
    const int ch0 = (blockIdx.x >> 1) * CH;
    const int H = a.H, b = blockIdx.y / H, h = blockIdx.y - b * H, tid = threadIdx.x, lane = tid & 63;
    const int index = lane < a.A ? a.accepted[b * a.A + lane] : -1;
    const int n = max(0, c.seq_lens[b]), n_rest = n % kRest, flushed = n - n_rest;
    const int count = accepted_count(index, a.T, n, c.max_seq_len);
    if (count == 0) return;
    unsigned short *rest = reinterpret_cast<unsigned short *>(is_v ? c.restv : c.restk) + ((int64_t)b * kRest * H + h) * D + ch0;
    const unsigned short *draft = reinterpret_cast<const unsigned short *>(is_v ? c.v : c.k) + ((int64_t)b * a.T * H + h) * D + ch0;
    const int64_t row = (int64_t)H * D;
    const int total = n_rest + count;
    const bool flush = total >= kRest;
    // the grown rest buffer: old rows only where they are flushed.  Its new rows go back to the rest buffer unless they are flushed,
    // those behind the flush to its front.  (Rows read here are written below, behind the barrier.)
    const int ch = tid % LANES * 4;
    for (int r0 = flush ? 0 : n_rest; r0 < total; r0 += 256 / LANES) {
        const int r = r0 + tid / LANES;
        const int from = __shfl(index, max(0, min(r - n_rest, 63)));
        if (r < total) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(r < n_rest ? rest + r * row + ch : draft + from * row + ch);
            *reinterpret_cast<u32 *>(&tile[r * PITCH + ch]) = w.x;
            *reinterpret_cast<u32 *>(&tile[r * PITCH + ch + 2]) = w.y;
        }
    }
    __syncthreads();
    uint8_t *colmax = (is_v ? c.v_max : c.k_max) + ((int64_t)b * H + h) * D + ch0;
    if (tid < CH) {
        int mx = colmax[tid];
        for (int r = n_rest; r < total; ++r) mx = max(mx, (tile[r * PITCH + tid] >> 10) & 31);
        colmax[tid] = (uint8_t)mx;
    }
    const int first = flush ? kRest : n_rest, shift = flush ? kRest : 0;
    for (int r0 = first; r0 < total; r0 += 256 / LANES) {
        const int r = r0 + tid / LANES;
        if (r < total) {
            const u32x2 w = {*reinterpret_cast<const u32 *>(&tile[r * PITCH + ch]), *reinterpret_cast<const u32 *>(&tile[r * PITCH + ch + 2])};
            *reinterpret_cast<u32x2 *>(rest + (r - shift) * row + ch) = w;
        }
    }
    if (!flush) return;
    const int64_t bh = (int64_t)b * H + h;
    // four elements side by side in a plane at a time: four channels of a token (values), four tokens of a channel (keys)
    for (int id = tid; id < kRest * CH / 4; id += 256) {
        const int r = is_v ? id / LANES : id % (kRest / 4) * 4, d = is_v ? id % LANES * 4 : id / (kRest / 4), next = is_v ? 1 : PITCH;
        const unsigned short *e = &tile[r * PITCH + d];
        const u32 w0 = e[0], w1 = e[next], w2 = e[2 * next], w3 = e[3 * next];
        const int64_t at = is_v ? (bh * c.max_seq_len + flushed + r) * D + ch0 + d
                                : ((bh * c.n_max_blocks + flushed / c.k_block) * D + ch0 + d) * c.k_block + flushed % c.k_block + r;
        *reinterpret_cast<u32 *>((is_v ? c.v_first_8 : c.k_first_8) + at) = (w0 >> 8) | (w1 & 0xFF00u) | (w2 & 0xFF00u) << 8 | (w3 & 0xFF00u) << 16;
        *reinterpret_cast<unsigned short *>((is_v ? c.v_mid_4 : c.k_mid_4) + at / 2) =
            (unsigned short)((w0 & 0xF0) | ((w1 >> 4) & 15) | (w2 & 0xF0) << 8 | ((w3 >> 4) & 15) << 8);
        *reinterpret_cast<unsigned short *>((is_v ? c.v_last_4 : c.k_last_4) + at / 2) =
            (unsigned short)((w0 & 15) << 4 | (w1 & 15) | (w2 & 15) << 12 | (w3 & 15) << 8);
    }
}

// The lengths, once every workgroup of the launches before has read them.
constexpr int kLensLayers = 240;
struct CommitLens {
    int *seq_lens[kLensLayers];
    int capacity[kLensLayers];
    const int *accepted;
    int T, A;
};
static_assert(sizeof(CommitLens) <= 4096, "kernel arguments");
__global__ __launch_bounds__(64) void tree_commit_lens_kernel(CommitLens a) {
    const int b = blockIdx.x, lane = threadIdx.x;
    const int index = lane < a.A ? a.accepted[b * a.A + lane] : -1;
    int *lens = a.seq_lens[blockIdx.y];
    const int n = max(0, lens[b]), count = accepted_count(index, a.T, n, a.capacity[blockIdx.y]);
    if (lane == 0) lens[b] = n + count;
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

// How a call is cut up: the rows of a KV head into groups of 32, 64, 128 or 256 (4, 2, 1 or 1 parts), the planes into splits of whole rounds.
struct TreePlan {
    int parts, row_tile, tokens, groups, splits, own_tail;
};
static TreePlan tree_plan(int bsz, int n_kv_heads, int head_dim, int rows, int bound) {
    TreePlan p;
    p.parts = rows > 64 ? 1 : (rows > 32 ? 2 : 4);
    p.tokens = p.parts == 4 ? 128 : p.parts * (head_dim == 256 ? 32 : 64);
    // 512 threads share a round's planes, loaded and unpacked once, where there are more than 128 rows: 4 x 16384 tokens x 8 KV heads, 132 rows 98 to
    // 101 us against 110 with 256 threads, 192 99 to 101 against 109 to 112, 256 103 to 107 against 114 to 117, 272 169 against 191, 512 182 to 186
    // against 199; 8 x 4096 x 4, 136 rows 37.3 against 39.8, 256 42.5 against 43.7.  (head_dim 256: the registers of a wave, two to a SIMD, do not
    // hold it; 64: too few planes a round to share.)
    p.row_tile = head_dim == 128 && rows > 128 ? 256 : 128 / p.parts;
    p.groups = (rows + p.row_tile - 1) / p.row_tile;
    const int flushed = bound / kRest * kRest, rounds = (flushed + p.tokens - 1) / p.tokens;
    const int64_t units = (int64_t)bsz * n_kv_heads * p.groups;
    // Workgroups in one round of the chip: two a compute unit, one where a workgroup takes the registers of both.  16 drafts x 4 heads a KV
    // head over 8 sequences of 4075 to 8150 tokens: 58 us with 512, 64 with 384, 66 with 256; of 8192 each 76, 72 and 73 (more sums
    // to join).  With head_dim 64 the sums weigh more beside the planes: 8 drafts x 4 heads over 4 x 16384 tokens 41 us with 512, 34 with 384.
    const int aim = head_dim == 256 || p.row_tile == 256 ? 256 : (head_dim == 64 && p.parts > 1 ? 384 : 512);
    int64_t want = (aim + units - 1) / units;
    if (want > rounds) want = rounds;
    if (want < 1) want = 1;
    // the tails get workgroups of their own while there are compute units without one
    p.own_tail = rounds > 0 && units * (want + 1) <= 256;
    p.splits = (int)(want + p.own_tail) * bsz;
    return p;
}

template <int D, int KB>
static void launch_tree(const TreeArgs &a, const TreePlan &p, bool cap, hipStream_t st) {
    const dim3 grid((u32)(((int64_t)p.splits * a.c.n_kv_heads + 7) / 8 * 8 * p.groups));
    const bool alibi = a.slopes != nullptr;
    constexpr int BN = D == 256 ? 32 : 64;
#define AKV_TREE(PARTS, BN, THREADS, CAP, ALIBI) hipLaunchKernelGGL((tree_kernel<D, KB, PARTS, BN, THREADS, CAP, ALIBI>), grid, dim3(THREADS), 0, st, a)
#define AKV_TREE_PARTS(PARTS, BN, THREADS)                                                                                         \
    do {                                                                                                                  \
        if (cap) { if (alibi) AKV_TREE(PARTS, BN, THREADS, true, true); else AKV_TREE(PARTS, BN, THREADS, true, false); }                   \
        else { if (alibi) AKV_TREE(PARTS, BN, THREADS, false, true); else AKV_TREE(PARTS, BN, THREADS, false, false); }                     \
    } while (0)
    if (p.parts == 4) AKV_TREE_PARTS(4, 32, 256);
    else if (p.parts == 2) AKV_TREE_PARTS(2, BN, 256);
    else if (p.row_tile == 128) AKV_TREE_PARTS(1, BN, 256);
    else if constexpr (D == 128) AKV_TREE_PARTS(1, BN, 512);
#undef AKV_TREE_PARTS
#undef AKV_TREE
    hipLaunchKernelGGL(tree_combine_kernel<D>, dim3((a.rows + 1024 / D - 1) / (1024 / D), a.c.n_kv_heads, a.c.bsz), dim3(256), 0, st, a);
}

}  // namespace akv

extern "C" size_t akv_tree_attention_workspace_bytes(int bsz, int n_q_heads, int n_kv_heads, int head_dim, int n_drafts, int len_bound) {
    if (bsz < 1 || n_q_heads < 1 || n_kv_heads < 1 || n_q_heads % n_kv_heads || head_dim < 1 || n_drafts < 1 || n_drafts > 64 || len_bound < 0) return 0;
    const int rows = n_q_heads / n_kv_heads * n_drafts;
    const akv::TreePlan p = akv::tree_plan(bsz, n_kv_heads, head_dim, rows, len_bound);
    return (size_t)n_kv_heads * p.splits * rows * (head_dim + 2) * sizeof(float) + (size_t)bsz * 2 * sizeof(int);
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
    const akv::TreePlan p = akv::tree_plan(layer->bsz, layer->n_kv_heads, layer->head_dim, a.rows, len_bound);
    a.log_tokens = __builtin_ctz((unsigned)p.tokens); a.splits = p.splits; a.own_tail = p.own_tail;
    a.shares = reinterpret_cast<int *>(a.parts + (size_t)layer->n_kv_heads * p.splits * a.rows * (layer->head_dim + 2));
    AKV_REQUIRE(((int64_t)p.splits * layer->n_kv_heads + 8) * p.groups < (1ll << 31), "tree_attention: too many rows");
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
        AKV_REQUIRE((((uintptr_t)k[i] | (uintptr_t)v[i]) & 7) == 0, "tree_commit: k and v must be 8-byte aligned");
        AKV_REQUIRE(layers[i].bsz == layers[0].bsz && layers[i].n_kv_heads == layers[0].n_kv_heads && layers[i].head_dim == layers[0].head_dim,
                    "tree_commit: layer %d has another shape than layer 0", i);
        for (int j = 0; j < i; ++j)
            AKV_REQUIRE(layers[i].seq_lens != layers[j].seq_lens, "tree_commit: layers %d and %d share their lengths", j, i);
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int streams = layers[0].bsz * layers[0].n_kv_heads;
    for (int first = 0; first < n_layers; first += akv::kCommitLayers) {
        const int count = n_layers - first < akv::kCommitLayers ? n_layers - first : akv::kCommitLayers;
        akv::CommitArgs a;
        for (int i = 0; i < count; ++i) {
            const akv_cache_layer &c = layers[first + i];
            a.c[i] = {c.k_first_8, c.k_mid_4, c.k_last_4, c.v_first_8, c.v_mid_4, c.v_last_4, c.k_exp_column_max, c.v_exp_column_max, c.restk, c.restv,
                      c.seq_lens, k[first + i], v[first + i], c.n_max_blocks, c.max_seq_len, c.k_block};
        }
        a.accepted = accepted;
        a.T = n_drafts;
        a.A = n_accepted;
        a.H = layers[0].n_kv_heads;
        const dim3 grid(2 * layers[0].head_dim / 64, streams, count);
        if (layers[0].head_dim == 64) hipLaunchKernelGGL(akv::tree_commit_kernel<64>, grid, dim3(256), 0, st, a);
        else if (layers[0].head_dim == 128) hipLaunchKernelGGL(akv::tree_commit_kernel<128>, grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(akv::tree_commit_kernel<256>, grid, dim3(256), 0, st, a);
    }
    for (int first = 0; first < n_layers; first += akv::kLensLayers) {
        const int count = n_layers - first < akv::kLensLayers ? n_layers - first : akv::kLensLayers;
        akv::CommitLens a;
        for (int i = 0; i < count; ++i) {
            a.seq_lens[i] = layers[first + i].seq_lens;
            a.capacity[i] = layers[first + i].max_seq_len;
        }
        a.accepted = accepted;
        a.T = n_drafts;
        a.A = n_accepted;
        hipLaunchKernelGGL(akv::tree_commit_lens_kernel, dim3(layers[0].bsz, count), dim3(64), 0, st, a);
    }
    return akv::check_launch("tree_commit");
}
