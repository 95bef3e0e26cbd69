// Prompt attention, and the attention weight that prompt tokens received.
//
//   s_ij = cap(scale q_i . k_j) - slope_h |i - j|,   cap(x) = c tanh(x / c)
//   o_i  = sum_j softmax_j(s_ij) v_j,   lse_i = log sum_j exp(s_ij)
// over the tokens j that row i sees: i, j < length, j <= i or j < prefix, same document (ids >= 0).  A row that sees
// nothing gives zeros and lse = -inf.
#include "akv_attention.h"

namespace akv {

struct PromptArgs {
    const uint8_t *q, *k, *v;                 // fp16
    int64_t q_b, q_s, q_h, k_b, k_s, k_h, v_b, v_s, v_h;   // strides in bytes
    const float *slopes;                      // [Hq] or null
    const int *lens, *prefix;                 // [B] or null
    const int *docs;                          // [B, S] or null
    const int *order;                         // [B, row tiles]: with documents, the row tiles in the order in which they start
    const u32x4 *doc_tiles;                   // [B, tiles of the K/V tile's tokens]: {smallest id, largest id, all the same, 0}
    int B, S, Hq, Hkv, G;
    ScoreForm form;
    float neg_slope_unit;                     // -log2 e
};

constexpr int kTileMin = 32;    // tokens of a K/V tile, and of a range of documents: 64, or 32 for head_dim 256

constexpr int kMaxSorted = 4096;   // K/V tiles up to which the row tiles of a sequence are put in order of their work

// One workgroup per sequence.  The range of documents of every K/V tile; and the row tiles (ROWS rows each) in order of the
// number of K/V tiles they have to look at, most first: workgroups start in that order, and a long one that starts last is what
// the others wait for (8192 tokens in 3 documents, 32 heads x 128, capped, eight orders of the documents: calls of 306 to 327 us in this order, 303
// to 365 by rows; 12 us of a call are this kernel, whose one workgroup does ranges, costs and ranks in turn).
__global__ __launch_bounds__(1024) void doc_tiles_kernel(const int *__restrict__ docs, const int *__restrict__ lens, const int *__restrict__ prefix_lens,
                                                         u32x4 *__restrict__ out, int *__restrict__ order, int S, int tiles, int tile, int row_tiles, int rows) {
    __shared__ u32 lo_s[kMaxSorted], hi_s[kMaxSorted];
    __shared__ int cost_s[kMaxSorted];
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = wave_index();
    const int n = lens ? max(0, min(lens[b], S)) : S, prefix = prefix_lens ? min(prefix_lens[b], n) : 0;
    const bool sorted = tiles <= kMaxSorted && row_tiles <= kMaxSorted;
    for (int t = wave; t < tiles; t += 16) {
        const int j = t * tile + lane;
        const bool in = lane < tile && j < n;
        const int d = in ? docs[(int64_t)b * S + j] : -1;
        const bool real = d >= 0;
        const u32 lo = wave_min_u32(real ? (u32)d : 0x7fffffffu);
        const u32 hi = ~wave_min_u32(real ? ~(u32)d : 0xffffffffu);   // largest id; 0 where there is none (then lo > hi)
        const bool same = __all(!in || (u32)d == lo) && lo <= hi;
        if (lane == 0) {
            out[(int64_t)b * tiles + t] = u32x4{lo, hi, same ? 1u : 0u, 0u};
            if (sorted) {
                lo_s[t] = lo;
                hi_s[t] = hi;
            }
        }
    }
    int *my_order = order + (int64_t)b * row_tiles;
    if (!sorted) {
        for (int r = threadIdx.x; r < row_tiles; r += 1024) my_order[r] = row_tiles - 1 - r;
        return;
    }
    __syncthreads();
    for (int r = wave; r < row_tiles; r += 16) {
        const int last = min(r * rows + rows, n) - 1, end = (max(last + 1, prefix) + tile - 1) / tile;
        u32 lo = 0xffffffffu, hi = 0;
        for (int t = r * rows / tile; t <= last / tile; ++t) {
            lo = min(lo, lo_s[t]);
            hi = max(hi, lo_s[t] <= hi_s[t] ? hi_s[t] : 0u);
        }
        int cost = 0;
        if (last >= r * rows)
            for (int t = lane; t < end; t += 64) cost += lo_s[t] <= hi && hi_s[t] >= lo && lo_s[t] <= hi_s[t] ? 1 : 0;
        cost = wave_sum_i32(cost);
        if (lane == 0) cost_s[r] = cost;
    }
    __syncthreads();
    for (int r = threadIdx.x; r < row_tiles; r += 1024) {
        const int mine = cost_s[r];
        int rank = 0;
        for (int k = 0; k < row_tiles; ++k) rank += cost_s[k] > mine || (cost_s[k] == mine && k > r) ? 1 : 0;
        my_order[rank] = r;
    }
}

// The K/V tiles a workgroup has to look at, in order.  Without documents all of [0, end); with them those whose range of
// ids meets the rows' (64 ranges per look).
template <bool DOCS>
struct TileWalk {
    const u32x4 *ranges = nullptr;
    u32 lo = 0, hi = 0;
    bool rows_same = false;
    int end = 0, next_tile = 0, base = -64;
    unsigned long long live = 0, same = 0;
    bool cur_same = true;       // every visible pair of (rows, last returned tile) is of one document

    __device__ __forceinline__ int next() {
        if constexpr (!DOCS) {
            return next_tile < end ? next_tile++ : -1;
        } else {
            while (live == 0) {
                base += 64;
                if (base >= end) return -1;
                const int t = base + (int)(threadIdx.x & 63);
                u32x4 r = {1u, 0u, 0u, 0u};
                if (t < end) r = ranges[t];
                live = __ballot(t < end && r.x <= hi && r.y >= lo && r.x <= r.y);
                same = __ballot(r.z != 0 && rows_same && r.x == lo);
            }
            const int i = __builtin_ctzll(live);
            live &= live - 1;
            cur_same = (same >> i) & 1;
            return base + i;
        }
    }
};

// A workgroup's share of the work: query tile, query head, sequence.  Blocks are dealt out to the 8 XCDs in turn; the
// query heads of one KV head, which read the same keys and values, are kept on one XCD (its L2), and the tiles with the
// most tokens to look at (the last ones, under a causal mask) come first.
__device__ __forceinline__ void prompt_block(int id, int n_tiles, int B, int Hkv, int G, int &qt, int &hq, int &b) {
    const int streams = B * Hkv;
    int stream, rest;
    if (streams % 8 == 0) {
        const int per = streams / 8, x = id & 7, i = id >> 3;
        stream = (i / G) % per * 8 + x;
        rest = i / (G * per) * G + i % G;
    } else {
        stream = (id / G) % streams;
        rest = id / (G * streams) * G + id % G;
    }
    qt = n_tiles - 1 - rest / G;
    b = stream / Hkv;
    hq = (stream - b * Hkv) * G + rest % G;
}

// One pass over the tokens with a running maximum and sum in 32 bits (the sum is rescaled only when the maximum has grown by 2^8); scores are
// computed transposed, so that a lane owns a query row and its probabilities are the second product's operand where they are, rounded
// to fp16 for it (2^-11 of each, or 2^-32 of the row's largest; its sums are in 32 bits).  Bound by the arithmetic.  8192 tokens, causal, of the
// 1251 TFLOP/s that a large fp16 matrix product reaches here: 32 heads over 8 x 128 577 us, 953 TFLOP/s; x 64 334 us, 824 TFLOP/s, where a score's
// scaling and exponential weigh twice as much beside its products; 16 heads over 4 x 256 921 us, 597 TFLOP/s, a wave to a SIMD (capped 1106 us).
// grid n_tiles * Hq * B, 256 threads.  K and V tiles of BN tokens go through LDS, two buffers, filled by asynchronous loads: the
// next tiles are in flight while these are computed, one barrier a round.  PARTS == 1: 128 query rows of one head, 32 a wave, all
// on the same tile.  PARTS == 2: 64 rows, two waves on every other tile each, their sums joined at the end: half the rounds for a
// row, for calls whose longest rows, not their number, decide how long they take.
template <int D, int BN, int PARTS, bool CAP, bool ALIBI, bool DOCS>
__global__ __launch_bounds__(256, D == 256 || D * PARTS == 256 ? 1 : (D == 64 && PARTS == 1 && !DOCS ? 3 : 2)) void prefill_kernel(PromptArgs a, uint8_t *__restrict__ out, float *__restrict__ lse,
                                                                                            int n_tiles, int fill) {
    constexpr int CPR = D / 8;                       // 16-byte chunks of a token
    constexpr int LPT = BN * CPR / 256;              // chunks a thread loads per tile and side
    constexpr int TB = BN / 32;
    constexpr int kSide = BN * D * 2;
    constexpr int ROWS = 128 / PARTS, WAVES = 4 / PARTS;      // rows of the workgroup, waves per part
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2][PARTS][2][kSide];
    __shared__ int odd_tile[PARTS];                  // the last tile in which a wave found a value that is not finite
    const int lane = threadIdx.x & 63, wave = wave_index(), half = lane >> 5, part = wave / WAVES, tid = threadIdx.x & (64 * WAVES - 1);
    int qt, hq, b;
    prompt_block(blockIdx.x, n_tiles, a.B, a.Hkv, a.G, qt, hq, b);
    const int hkv = hq / a.G;
    if constexpr (DOCS) qt = a.order[(int64_t)b * n_tiles + n_tiles - 1 - qt];
    const int n = a.lens ? max(0, min(a.lens[b], a.S)) : a.S;
    const int prefix = a.prefix ? min(a.prefix[b], n) : 0;
    const int row0 = qt * ROWS, i0 = row0 + (wave % WAVES) * 32, i = i0 + (lane & 31);

    f32x16 o[D / 32];
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[cb][r] = 0.f;
    RowState st;
    OddValues<D> odd;

    if (row0 < n) {
        f16x8 qf[D / 16];
        const uint8_t *qp = a.q + b * a.q_b + (int64_t)min(i, n - 1) * a.q_s + hq * a.q_h;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *reinterpret_cast<const f16x8 *>(qp + (2 * ks + half) * 16);
        const int my_doc = DOCS ? a.docs[(int64_t)b * a.S + min(i, n - 1)] : 0;
        const float neg_slope = ALIBI ? a.slopes[hq] * -kLog2e : 0.f;
        const int last_row = min(row0 + ROWS - 1, n - 1);
        TileWalk<DOCS> walk;
        walk.end = (max(last_row + 1, prefix) + BN - 1) / BN;
        if constexpr (DOCS) {
            walk.ranges = a.doc_tiles + (int64_t)b * ((a.S + BN - 1) / BN);
            walk.lo = 0xffffffffu;
            walk.hi = 0;
            walk.rows_same = true;
            u32 first = 0;
#pragma unroll
            for (int s = 0; s < ROWS / BN; ++s) {
                if (row0 + s * BN > last_row) continue;
                const u32x4 r = walk.ranges[row0 / BN + s];
                if (s == 0) first = r.x;
                walk.lo = min(walk.lo, r.x);
                walk.hi = max(walk.hi, r.x <= r.y ? r.y : 0u);
                walk.rows_same = walk.rows_same && r.z && r.x == first;
            }
        }
        const uint8_t *kp = a.k + b * a.k_b + hkv * a.k_h, *vp = a.v + b * a.v_b + hkv * a.v_h;
        // piece c * 256 + thread of a tile lies at that place in LDS: row piece / CPR, and the chunk that the layout puts there
        const int my_row = threadIdx.x / CPR;
        LaneBytes<D> at;
        const u32 lds0 = lds_address(&lds[0][0][0][0]) + wave * 1024;
        auto request = [&](int t, int slot) {
            const int j0 = t * BN, rows = min(BN, n - j0);
            const auto rk = make_rsrc(kp + (int64_t)j0 * a.k_s, (u32)((rows - 1) * a.k_s + D * 2));
            const auto rv = make_rsrc(vp + (int64_t)j0 * a.v_s, (u32)((rows - 1) * a.v_s + D * 2));
#pragma unroll
            for (int c = 0; c < LPT; ++c) {
                // behind the sequence's end its last token stands in for the missing ones: no row sees them
                const int r = my_row + c * (256 / CPR), row = min(r, rows - 1), ch = ((int)threadIdx.x % CPR ^ tile_swizzle<D>(r)) << 4;
                load_to_lds(rk, lds0 + slot * (2 * kSide) + c * 4096, (int)(row * a.k_s) + ch);
                load_to_lds(rv, lds0 + slot * (2 * kSide) + kSide + c * 4096, (int)(row * a.v_s) + ch);
            }
        };
        if (threadIdx.x < PARTS) odd_tile[threadIdx.x] = -1;
        // the tiles of this round and of the next; t[0] < 0: none are left
        int t[PARTS], t_next[PARTS], buf = 0;
        bool same[PARTS], same_next[PARTS];
        int token_doc = 0, doc_next = 0;               // document of token `lane` of this wave's tile, where rows are told apart by it
        auto fetch = [&](int into) {
#pragma unroll
            for (int s = 0; s < PARTS; ++s) {
                t_next[s] = s > 0 && t_next[s - 1] < 0 ? -1 : walk.next();
                same_next[s] = walk.cur_same;
            }
            if (into < 0) return;
#pragma unroll
            for (int s = 0; s < PARTS; ++s)
                if (t_next[s] >= 0) {
                    request(t_next[s], into * PARTS + s);
                    if constexpr (DOCS)
                        if (s == part && !same_next[s]) doc_next = a.docs[(int64_t)b * a.S + min(t_next[s] * BN + lane, n - 1)];
                }
        };
        fetch(0);
        while (t_next[0] >= 0) {
#pragma unroll
            for (int s = 0; s < PARTS; ++s) {
                t[s] = t_next[s];
                same[s] = same_next[s];
            }
            wait_tile();
            token_doc = doc_next;
            fetch(buf ^ 1);
            const int my_t = PARTS == 1 || part == 0 ? t[0] : t[PARTS - 1];
            const bool my_same = PARTS == 1 || part == 0 ? same[0] : same[PARTS - 1];
            const int j0 = my_t * BN;
            uint8_t *kt = lds[buf][part][0], *vt = lds[buf][part][1];
            at.pin();
            // token 32 tb + 8 (r / 4) + r % 4 of the tile is seen if that number is at most lim
            const int lim = min(max(i, prefix - 1), n - 1) - j0 - 4 * half;
            const bool whole = j0 + BN <= n && my_same;      // no row misses tokens for their length or document
            const auto sees = [&](int c) {
                bool see = c <= lim;
                if constexpr (DOCS) {
                    const int d0 = __builtin_amdgcn_readlane(token_doc, c), d1 = __builtin_amdgcn_readlane(token_doc, c + 4);
                    see = see && (my_same || ((half ? d1 : d0) == my_doc && my_doc >= 0));
                }
                return see;
            };
            bool edge = false;
#pragma unroll
            for (int s = 0; s < PARTS; ++s) edge = edge || (t[s] >= 0 && (!same[s] || t[s] * BN + BN > n || t[s] * BN + BN - 1 > max(row0, prefix - 1)));
            if (edge) {
                if (my_t >= 0 && share_nonfinite<D, BN, 64 * WAVES>(vt, tid)) odd_tile[part] = my_t;
                lds_barrier();
                bool found = odd_tile[0] == t[0];
                if constexpr (PARTS == 2) found = found || (t[1] >= 0 && odd_tile[1] == t[1]);
                if (found) {
                    if (my_t >= 0) {
                        u32 seen = 0;
#pragma unroll
                        for (int c = 0; c < TB * 16; ++c) seen |= sees((c >> 4) * 32 + 8 * ((c & 15) >> 2) + (c & 3)) ? 1u << c : 0u;
                        note_nonfinite<D, BN>(odd, vt, at, seen);
                    }
                    lds_barrier();
                    if (my_t >= 0) zero_nonfinite_tile<D, BN, 64 * WAVES>(vt, tid);
                    lds_barrier();
                }
            }
            const int wave_last = min(i0 + 31, n - 1);
            if (my_t >= 0 && i0 < n && (j0 <= wave_last || j0 < prefix)) {
                f32x16 x[TB];
                tile_scores<D, BN>(x, kt, at, qf);
                const float factor = modify_block<CAP, TB>(x, a.form);
                float shift = 0.f;
                if constexpr (ALIBI) {
                    const float gap0 = (float)(j0 + 4 * half - i), s = neg_slope / factor;
                    if (j0 >= prefix || j0 + BN - 1 <= i0) {
                        // every token that is seen lies before its row: the distance is linear in the token, and the row's part of
                        // it is the same for the whole tile
                        shift = -neg_slope * gap0;
#pragma unroll
                        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                            for (int r = 0; r < 16; ++r) x[tb][r] = fmaf(-s, (float)(tb * 32 + 8 * (r >> 2) + (r & 3)), x[tb][r]);
                    } else {
#pragma unroll
                        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                            for (int r = 0; r < 16; ++r) x[tb][r] = fmaf(s, fabsf(gap0 + (float)(tb * 32 + 8 * (r >> 2) + (r & 3))), x[tb][r]);
                    }
                }
                if (!whole || j0 + BN - 1 > max(i0, prefix - 1)) {
#pragma unroll
                    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[tb][r] = sees(tb * 32 + 8 * (r >> 2) + (r & 3)) ? x[tb][r] : kNegInf;
                }
                f16x8 p[TB][2];
                tile_softmax<D, BN>(x, factor, shift, st, o, p);
                tile_output<D, BN>(o, vt, at, p);
            }
            buf ^= 1;
        }
    }

    float l = halves_sum(st.l);
    if constexpr (PARTS == 2) {
        // the second part's sums through LDS, register by register (lane l's words lie next to lane l + 1's), into the first part's
        lds_barrier();
        float *box = reinterpret_cast<float *>(&lds[0][0][0][0]) + (wave % WAVES) * (64 * (D / 2 + 2 + D / 32)) + lane;
        static_assert(WAVES * 64 * (D / 2 + 2 + D / 32) * 4 <= sizeof(lds), "the sums of a part fit into the tiles' memory");
        if (part == 1) {
#pragma unroll
            for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
                for (int r = 0; r < 16; ++r) box[(cb * 16 + r) * 64] = o[cb][r];
            box[(D / 2) * 64] = st.m;
            box[(D / 2 + 1) * 64] = l;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int w = 0; w < D / 64; ++w) box[(D / 2 + 2 + s * (D / 64) + w) * 64] = __uint_as_float(odd.hit[s][w]);
        }
        lds_barrier();
        if (part == 1) return;
        const float m1 = box[(D / 2) * 64], m = fmaxf(st.m, m1);
        const float f0 = st.m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(st.m - m), f1 = m1 == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m1 - m);
        l = l * f0 + box[(D / 2 + 1) * 64] * f1;       // (zero times an undefined sum is undefined)
        st.m = m;
#pragma unroll
        for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[cb][r] = fmaf(box[(cb * 16 + r) * 64], f1, o[cb][r] * f0);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int w = 0; w < D / 64; ++w) odd.hit[s][w] |= __float_as_uint(box[(D / 2 + 2 + s * (D / 64) + w) * 64]);
    }
    if (i >= a.S) return;
    if (i >= n && !fill) return;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);    // (an undefined sum stays undefined)
    uint8_t *op = out + (((int64_t)b * a.S + i) * a.Hq + hq) * (D * 2);
    if (i >= n) {
#pragma unroll
        for (int c = 0; c < CPR / 2; ++c) *reinterpret_cast<u32x4 *>(op + (2 * c + half) * 16) = u32x4{0u, 0u, 0u, 0u};
    } else {
        if (odd.any()) odd.add(o);
#pragma unroll
        for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const u32x2 w = {pack_f16(o[cb][4 * g] * inv, o[cb][4 * g + 1] * inv), pack_f16(o[cb][4 * g + 2] * inv, o[cb][4 * g + 3] * inv)};
                *reinterpret_cast<u32x2 *>(op + (cb * 32 + 8 * g + 4 * half) * 2) = w;
            }
    }
    if (lse != nullptr && half == 0)
        lse[((int64_t)b * a.Hq + hq) * a.S + i] = i < n ? (l == 0.f ? kNegInf : (st.m - kLift + __builtin_amdgcn_logf(l)) * kLn2) : kNegInf;
}

// ---- the weight each token received -----------------------------------------------------------------------------------------------
// w_j = sum over the heads g of the group and the rows i of the window of exp(s_ij - lse_i).  A workgroup owns 128 tokens of one KV
// head, a wave 32 of them, whose keys stay in registers; the rows, head after head, stream past them through LDS, QR at a
// time, two buffers filled by asynchronous loads (rows read by their lanes straight from memory, 32 lines a request, kept the address
// units busy: 39 us at 2 x 8000 tokens, 64 rows of 32 heads over 8 x 128, 18 through LDS).  Its bound: 33 MB of keys (6.5 us) and, behind them
// because all workgroups start with their keys, 8.4 GFLOP with an exponential a score.  A lane sums its row's column of each product, and one
// reduction over the rows' lanes ends it.  No atomics: the order of a sum is fixed.
template <int D, bool CAP, bool ALIBI>
__global__ __launch_bounds__(256) void attention_weights_kernel(PromptArgs a, const float *__restrict__ lse, int window, float *__restrict__ w,
                                                                int64_t w_b, int64_t w_h, int add) {
    constexpr int QR = D == 256 ? 32 : 64, CPR = D / 8, kQ = QR * D * 2;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[128 * D * 2 > 2 * kQ ? 128 * D * 2 : 2 * kQ];       // the keys, then the rows
    const int lane = threadIdx.x & 63, wave = wave_index(), half = lane >> 5, col = lane & 31;
    const int hkv = blockIdx.y, b = blockIdx.z, jw = blockIdx.x * 128, j0 = jw + wave * 32;
    const int n = a.lens ? max(0, min(a.lens[b], a.S)) : a.S;
    const int prefix = a.prefix ? min(a.prefix[b], n) : 0;
    float sum[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[r] = 0.f;
    int first = window > 0 ? max(0, n - window) : 0;
    if (jw >= prefix) first = max(first, jw);           // rows before the tokens do not see them
    const int blocks = jw < n ? (n - first + QR - 1) / QR : 0, rounds = blocks * a.G;
    if (rounds > 0) {
        const u32 lds0 = lds_address(lds) + wave * 1024;
        const int my_row = threadIdx.x / CPR, my_chunk = threadIdx.x % CPR;
        // rows j .. j + ROWS - 1 of a [token, head] matrix to LDS at byte `at`, the last row in place of those at and beyond n
        auto bring = [&](const uint8_t *base, int64_t stride, int j, int rows_max, int at) {
            const int rows = min(rows_max, n - j);
            const auto rs = make_rsrc(base + (int64_t)j * stride, (u32)((rows - 1) * stride + D * 2));
            for (int c = 0; c < rows_max * CPR / 256; ++c) {
                const int r = my_row + c * (256 / CPR);
                load_to_lds(rs, lds0 + at + c * 4096, (int)(min(r, rows - 1) * stride) + ((my_chunk ^ tile_swizzle<D>(r)) << 4));
            }
        };
        bring(a.k + b * a.k_b + hkv * a.k_h, a.k_s, jw, 64, 0);
        if (jw + 64 < n) bring(a.k + b * a.k_b + hkv * a.k_h, a.k_s, jw + 64, 64, 64 * D * 2);
        wait_tile();
        f16x8 kf[D / 16];
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) kf[ks] = *reinterpret_cast<const f16x8 *>(lds + tile_byte<D>(wave * 32 + col, 2 * ks + half));
        int doc[16];
        if (a.docs) {
#pragma unroll
            for (int r = 0; r < 16; ++r) doc[r] = a.docs[(int64_t)b * a.S + min(j0 + 8 * (r >> 2) + 4 * half + (r & 3), n - 1)];
        }
        lds_barrier();
        float row_lse[QR / 32], lse_next[QR / 32];
        auto request = [&](int round, int buf) {
            const int g = round / blocks, i0 = first + (round - g * blocks) * QR, hq = hkv * a.G + g;
            bring(a.q + b * a.q_b + hq * a.q_h, a.q_s, i0, QR, buf * kQ);
#pragma unroll
            for (int tb = 0; tb < QR / 32; ++tb) lse_next[tb] = lse[((int64_t)b * a.Hq + hq) * a.S + min(i0 + tb * 32 + col, n - 1)];
        };
        request(0, 0);
        int at_q = tile_byte<D>(col, half);
        for (int round = 0; round < rounds; ++round) {
            wait_tile();
#pragma unroll
            for (int tb = 0; tb < QR / 32; ++tb) row_lse[tb] = lse_next[tb] * kLog2e;
            if (round + 1 < rounds) request(round + 1, (round + 1) & 1);
            const int g = round / blocks, i0 = first + (round - g * blocks) * QR;
            const float neg_slope = ALIBI ? a.slopes[hkv * a.G + g] * -kLog2e : 0.f;
            const uint8_t *qt = lds + (round & 1) * kQ;
            asm volatile("" : "+v"(at_q));
#pragma unroll
            for (int tb = 0; tb < QR / 32; ++tb) {
                const int ib = i0 + tb * 32, i = ib + col;
                if (ib >= n || (j0 > ib + 31 && j0 >= prefix) || j0 >= n) continue;
                f32x16 x;
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = 0.f;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks], *reinterpret_cast<const f16x8 *>(qt + tb * 32 * D * 2 + (at_q ^ (ks << 5))), x, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if constexpr (CAP) x[r] = fmaf(a.form.c1, tanh_f32(x[r] * a.form.c0), -row_lse[tb]);
                    else x[r] = fmaf(x[r], a.form.c0, -row_lse[tb]);
                    if constexpr (ALIBI) x[r] = fmaf(neg_slope, fabsf((float)(j0 + 4 * half + 8 * (r >> 2) + (r & 3) - i)), x[r]);
                }
                if (a.docs || ib + 32 > n || j0 + 32 > n || j0 + 31 > max(ib, prefix - 1)) {
                    const int lim = i < n ? min(max(i, prefix - 1), n - 1) - j0 - 4 * half : -1;
                    const int my_doc = a.docs ? a.docs[(int64_t)b * a.S + min(i, n - 1)] : 0;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const bool see = 8 * (r >> 2) + (r & 3) <= lim && (!a.docs || (doc[r] == my_doc && my_doc >= 0));
                        x[r] = see ? x[r] : kNegInf;
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) sum[r] += __builtin_amdgcn_exp2f(x[r]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float s = lane_group_sum<16>(sum[r]);
        const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(s), __float_as_uint(s), false, false);
        sum[r] = __uint_as_float(t[0]) + __uint_as_float(t[1]);
    }
    if (col == 0) {
        float *wp = w + b * w_b + hkv * w_h;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = j0 + 8 * (r >> 2) + 4 * half + (r & 3);
            if (j >= a.S) continue;
            if (add) {
                if (j < n) wp[j] += sum[r];
            } else {
                wp[j] = sum[r];
            }
        }
    }
}

static int prompt_args(PromptArgs &a, const akv_prompt_desc *d, const char *what) {
    AKV_REQUIRE(d != nullptr, "%s: null descriptor", what);
    AKV_REQUIRE(d->q && d->k, "%s: null pointer", what);
    AKV_REQUIRE(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, "%s: head_dim %d: 64, 128 or 256", what, d->head_dim);
    AKV_REQUIRE(d->bsz >= 1 && d->seqlen >= 1 && d->seqlen <= (1 << 30) && d->n_kv_heads >= 1 && d->n_q_heads >= 1 && d->n_q_heads % d->n_kv_heads == 0,
                "%s: bsz %d, seqlen %d, heads %d / %d", what, d->bsz, d->seqlen, d->n_q_heads, d->n_kv_heads);
    AKV_REQUIRE(d->bsz <= 65535 && d->n_kv_heads <= 65535, "%s: at most 65535 sequences and KV heads", what);
    AKV_REQUIRE(d->scale > 0.f && d->scale < 1e30f, "%s: scale %g must be positive and finite", what, d->scale);
    AKV_REQUIRE(d->softcap >= 0.f && d->softcap < 1e30f, "%s: softcap %g must be zero (off) or positive and finite", what, d->softcap);
    const int64_t *strides[3] = {d->q_stride, d->k_stride, d->v_stride};
    const void *ptrs[3] = {d->q, d->k, d->v};
    for (int t = 0; t < 3; ++t) {
        if (ptrs[t] == nullptr) continue;
        AKV_REQUIRE(((uintptr_t)ptrs[t] & 15) == 0, "%s: q, k and v must be 16-byte aligned", what);
        for (int i = 0; i < 3; ++i)
            AKV_REQUIRE(strides[t][i] >= 0 && strides[t][i] % 8 == 0, "%s: strides must be multiples of 8 elements and not negative", what);
        AKV_REQUIRE(strides[t][1] < (1 << 24), "%s: a token stride of %lld elements: below 2^24", what, (long long)strides[t][1]);
    }
    a.q = d->q; a.k = d->k; a.v = d->v;
    a.q_b = d->q_stride[0] * 2; a.q_s = d->q_stride[1] * 2; a.q_h = d->q_stride[2] * 2;
    a.k_b = d->k_stride[0] * 2; a.k_s = d->k_stride[1] * 2; a.k_h = d->k_stride[2] * 2;
    a.v_b = d->v_stride[0] * 2; a.v_s = d->v_stride[1] * 2; a.v_h = d->v_stride[2] * 2;
    a.slopes = d->slopes; a.lens = d->seq_lens; a.prefix = d->prefix_lens; a.docs = d->documents;
    a.doc_tiles = nullptr;
    a.order = nullptr;
    a.B = d->bsz; a.S = d->seqlen; a.Hq = d->n_q_heads; a.Hkv = d->n_kv_heads; a.G = d->n_q_heads / d->n_kv_heads;
    a.form = score_form(d->scale, d->softcap);
    return AKV_OK;
}

// Whether a stretch of memory shares a byte with q, k or v.
static bool shares_inputs(const PromptArgs &a, int D, const void *p, int64_t bytes) {
    const auto with = [&](const uint8_t *x, int64_t b, int64_t s, int64_t h, int heads) {
        return x != nullptr && share_memory(p, bytes, x, (a.B - 1) * b + (a.S - 1) * s + (heads - 1) * h + D * 2);
    };
    return with(a.q, a.q_b, a.q_s, a.q_h, a.Hq) || with(a.k, a.k_b, a.k_s, a.k_h, a.Hkv) || with(a.v, a.v_b, a.v_s, a.v_h, a.Hkv);
}

// Two parts a row (64 rows a workgroup) pay while the workgroups of whole rows leave half of the compute units empty: 512 tokens x 32
// heads x 128 13.5 us against 15.2, x 16 heads x 256 24.3 against 33.4; with twice the rows 29.8 against 28.1 (fewer workgroups fit a compute
// unit, and each tile that is loaded serves half the rows).  And while the rounds they save outweigh the join of the parts.  Tokens
// and us of two parts / one, 8 to 128 heads alike, uncapped and capped: head_dim 64: 64 tokens 5.0 / 4.4 and 5.4 / 4.8, 128 5.2 / 5.7 and 5.5 /
// 6.5, 192 6.1 / 6.1 and 6.9 / 7.3, 256 6.2 / 7.5 and 7.0 / 9.0; 256: 64 tokens 10.6 / 9.0 and 10.8 / 9.8, 128 12.9 / 15.9 and 13.5 / 17.2, 256 16.7 /
// 21.4 and 17.9 / 24.5; 128: 128 tokens 7.9 / 7.4 and 8.2 / 8.3, 192 9.4 / 7.9 and 10.1 / 9.2, 256 9.7 / 9.9 and 10.4 / 11.6, 320 11.3 / 10.4 and 12.3 /
// 12.4, 384 11.6 / 12.5 and 12.6 / 15.2.
static int prompt_parts(const PromptArgs &a, int head_dim) {
    AKV_TUNE("AKV_TUNE_PROMPT_PARTS", forced);
    if (has_forced && (forced == 1 || forced == 2)) return forced;
    return a.S > (head_dim == 128 ? 256 : 64) && (int64_t)((a.S + 127) / 128) * a.Hq * a.B <= 128 ? 2 : 1;
}
template <int D, int BN, int PARTS>
static void launch_prefill(const PromptArgs &a, bool cap, uint8_t *out, float *lse, int fill, hipStream_t st) {
    const int n_tiles = (a.S + 128 / PARTS - 1) / (128 / PARTS);
    const dim3 grid((u32)((int64_t)n_tiles * a.Hq * a.B));
#define AKV_PREFILL(CAP, ALIBI, DOCS) \
    hipLaunchKernelGGL((prefill_kernel<D, BN, PARTS, CAP, ALIBI, DOCS>), grid, dim3(256), 0, st, a, out, lse, n_tiles, fill)
    if (a.docs) {
        if (cap) { if (a.slopes) AKV_PREFILL(true, true, true); else AKV_PREFILL(true, false, true); }
        else { if (a.slopes) AKV_PREFILL(false, true, true); else AKV_PREFILL(false, false, true); }
    } else {
        if (cap) { if (a.slopes) AKV_PREFILL(true, true, false); else AKV_PREFILL(true, false, false); }
        else { if (a.slopes) AKV_PREFILL(false, true, false); else AKV_PREFILL(false, false, false); }
    }
#undef AKV_PREFILL
}

}  // namespace akv

extern "C" size_t akv_prefill_attention_workspace_bytes(int bsz, int seqlen) {
    if (bsz < 1 || seqlen < 1) return 0;
    // ranges of documents, and an order of the row tiles (of at least 64 rows)
    return (size_t)bsz * (((size_t)seqlen + akv::kTileMin - 1) / akv::kTileMin * sizeof(u32x4) + ((size_t)seqlen + 63) / 64 * sizeof(int));
}

extern "C" int akv_prefill_attention(const akv_prompt_desc *desc, uint8_t *out, float *lse, int fill_padding, void *workspace,
                                     size_t workspace_bytes, akv_stream_t stream) {
    akv::PromptArgs a;
    const int rc = akv::prompt_args(a, desc, "prefill_attention");
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(a.v && out, "prefill_attention: null pointer");
    AKV_REQUIRE(((uintptr_t)out & 15) == 0, "prefill_attention: out must be 16-byte aligned");
    AKV_REQUIRE((int64_t)((a.S + 63) / 64) * a.Hq * a.B < (1ll << 31), "prefill_attention: too many rows");
    const size_t need = a.docs ? akv_prefill_attention_workspace_bytes(a.B, a.S) : 0;
    AKV_REQUIRE(!a.docs || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                "prefill_attention: documents need a 16-byte aligned workspace of %zu bytes, got %zu", need, workspace_bytes);
    const int64_t rows = (int64_t)a.B * a.S * a.Hq, out_bytes = rows * desc->head_dim * 2;
    AKV_REQUIRE(!akv::shares_inputs(a, desc->head_dim, out, out_bytes) && (lse == nullptr || (!akv::shares_inputs(a, desc->head_dim, lse, rows * 4) &&
                !akv::share_memory(out, out_bytes, lse, rows * 4))), "prefill_attention: out and lse must not overlap each other, q, k or v");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int parts = akv::prompt_parts(a, desc->head_dim);
    if (a.docs) {
        const int tile = desc->head_dim == 256 ? 32 : 64, tiles = (a.S + tile - 1) / tile;
        u32x4 *ranges = static_cast<u32x4 *>(workspace);
        int *order = reinterpret_cast<int *>(ranges + (size_t)a.B * tiles);
        a.doc_tiles = ranges;
        a.order = order;
        hipLaunchKernelGGL(akv::doc_tiles_kernel, dim3(a.B), dim3(1024), 0, st, a.docs, a.lens, a.prefix, ranges, order, a.S, tiles, tile, (a.S + 128 / parts - 1) / (128 / parts), 128 / parts);
    }
    const bool cap = desc->softcap > 0.f;
#define AKV_PREFILL_PARTS(D, BN)                                                                                              \
    do {                                                                                                                     \
        if (parts == 2) akv::launch_prefill<D, BN, 2>(a, cap, out, lse, fill_padding, st);                                    \
        else akv::launch_prefill<D, BN, 1>(a, cap, out, lse, fill_padding, st);                                               \
    } while (0)
    if (desc->head_dim == 64) AKV_PREFILL_PARTS(64, 64);
    else if (desc->head_dim == 128) AKV_PREFILL_PARTS(128, 64);
    else AKV_PREFILL_PARTS(256, 32);
#undef AKV_PREFILL_PARTS
    return akv::check_launch("prefill_attention");
}

extern "C" int akv_attention_weights(const akv_prompt_desc *desc, const float *lse, int window, float *weights, int64_t weights_stride_b,
                                     int64_t weights_stride_h, int add, akv_stream_t stream) {
    akv::PromptArgs a;
    const int rc = akv::prompt_args(a, desc, "attention_weights");
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(lse && weights, "attention_weights: null pointer");
    AKV_REQUIRE(window >= 0, "attention_weights: window %d must be 0 (every row) or positive", window);
    AKV_REQUIRE(weights_stride_h >= a.S || a.Hkv == 1, "attention_weights: rows of %lld weights for %d tokens", (long long)weights_stride_h, a.S);
    AKV_REQUIRE(akv::rows_apart(a.B, a.Hkv, a.S, weights_stride_b, weights_stride_h), "attention_weights: rows of weights share memory (strides %lld, %lld)",
                (long long)weights_stride_b, (long long)weights_stride_h);
    const int64_t span = akv::rows_span(a.B, a.Hkv, a.S, weights_stride_b, weights_stride_h);
    a.v = nullptr;      // (not read)
    AKV_REQUIRE(!akv::shares_inputs(a, desc->head_dim, weights, span) && !akv::share_memory(weights, span, lse, (int64_t)a.B * a.Hq * a.S * 4),
                "attention_weights: the weights must not overlap q, k or lse");
    const bool cap = desc->softcap > 0.f;
    const dim3 grid((a.S + 127) / 128, a.Hkv, a.B);
    const hipStream_t st = static_cast<hipStream_t>(stream);
#define AKV_WEIGHTS(D, CAP, ALIBI)                                                                                             \
    hipLaunchKernelGGL((akv::attention_weights_kernel<D, CAP, ALIBI>), grid, dim3(256), 0, st, a, lse, window, weights, weights_stride_b, \
                       weights_stride_h, add)
#define AKV_WEIGHTS_D(D)                                                                                    \
    do {                                                                                                    \
        if (cap) { if (a.slopes) AKV_WEIGHTS(D, true, true); else AKV_WEIGHTS(D, true, false); }            \
        else { if (a.slopes) AKV_WEIGHTS(D, false, true); else AKV_WEIGHTS(D, false, false); }              \
    } while (0)
    if (desc->head_dim == 64) AKV_WEIGHTS_D(64);
    else if (desc->head_dim == 128) AKV_WEIGHTS_D(128);
    else AKV_WEIGHTS_D(256);
#undef AKV_WEIGHTS_D
#undef AKV_WEIGHTS
    return akv::check_launch("attention_weights");
}
