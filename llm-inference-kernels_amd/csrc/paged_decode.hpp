// Decode attention over a paged cache for a batch of sequences of different
// lengths: one query per sequence,
//   out[b, h] = softmax_j(s(h, j)) V[j],  s = score of key j, over the live keys
// j < seq_lens[b] of the sequence's pages (the newest `window` of them), with the
// score options of ScoreOpts and a bias -slope[h] (pos - j).
//
// Bound: each K and V row is read once, 4 D bytes per 4 G D flops (G query heads
// per KV head), so the time is the cache's bytes over HBM's rate.
//
// Division of the work. The host does not know the lengths, so the grid is
// fixed and the workgroups divide the work themselves: the 32-token tiles of all
// (sequence, KV head, head chunk) slabs, one behind the other, are cut into equal
// shares of consecutive tiles, one per workgroup. A share may end one slab, hold
// whole ones and begin another: at most two of its pieces are parts of a slab,
// so the partial results need two slots per workgroup whatever the lengths are.
// The last of a slab's workgroups to arrive joins its parts in order (the parts,
// and so the bits, depend on the lengths of the whole batch, not on timing).
//
// A piece: four waves take its tiles in turn, each with its own running maximum
// and sum, and are joined through LDS. Products on 16x16x32 matrix instructions:
//   S^T = K q^T: A = 16 keys, B = the chunk's up to 16 heads: lane (g, c) gets the
//     scores of head c for tokens 4g .. 4g + 3 of each 16-token block;
//   O^T = V^T P^T: those scores are, unmoved, the B operand (k-slot 8g + e of the
//     32 is token 4g + e, or 16 + 4g + e - 4 from e = 4), and V's rows of the same
//     tokens, permuted in registers, the A operand (row m of product j is channel
//     VEC m + j, so a lane loads VEC neighbouring channels of a token at once).
// P enters as a pair hi + lo of 16-bit values (two products): its rounding then
// leaves 2^-22 (fp16) or 2^-16 (bf16) of each probability, less than the output's
// own; the second product is free beside the loads.
//
// Registers hold one tile: the next tile's keys are requested when the scores are
// computed, its values when their products are (two buffers spilled). Measured, GPU
// us: 64 sequences of 8192 tokens, 8 KV heads of 8 317 (6.8 TB/s); 32 of 30 .. 8000 in
// bf16 33.6 (5.0 TB/s); one of 50001, heads of 64, 23.4 (4.4 TB/s); 24 of 100 .. 12000
// in a window of 4096 23.1 (3.9 TB/s: small pages, a look-up per octet); one of 700 8.3,
// a chain of dependent reads (lengths, pages, keys, hand-off) behind the launch.
#pragma once

#include "paged_common.hpp"

namespace llmik {

constexpr int kPdWaves = 4;
constexpr int kPdThreads = kPdWaves * kWave;
constexpr int kPdPerCu = 2;       // workgroups per CU (3 spill: 32 ragged sequences 81 us instead of 33)

struct PagedDecodeParams {
    const uint16_t* q;
    uint16_t* out;
    PagedView c;
    ScoreOpts s;
    int n_heads, gqa, n_chunks, chunk_heads;   // query heads per KV head, their chunks, heads of a chunk (<= 16)
    int first;            // keys before this position are not this kernel's (the shared prefix)
    float* own_o;         // not null: a row's result goes, as sums, to the last of its own_parts
    float* own_ml;        //   parts [n_kv_heads, batch * gqa, own_parts, D] and (m, l), not to out
    int own_parts;
    float* part_o;        // [2 * workgroups, chunk_heads, D]
    float* part_ml;       // [2 * workgroups, chunk_heads, 2]
    uint32_t* counters;   // [workgroups], zero between calls
    int few_steps;        // workgroups that few tiles are spread over, one tile per wave
};

// kPieceUnits (llmik_internal.hpp) is a piece's overhead in units of a tile's time: see the shares.
constexpr int kUncutTiles = 12;   // a slab of so few tiles is not cut: three per wave cost less than a hand-off
constexpr int kEachTiles = 24;    // the longest slab where every workgroup takes one

// A sequence's length, its live keys [begin, end) and their 32-token tiles.
// Every sequence has one tile at least, so that its rows are written.
struct Keys {
    int len, begin, end, tiles;
};
__device__ __forceinline__ Keys keys_of(const PagedDecodeParams& p, int len) {
    Keys k;
    k.len = max(len, 0);
    k.end = min(k.len, p.c.capacity);
    k.begin = min(max(max(k.len - p.s.window, 0), p.first), k.end);
    k.tiles = max((k.end + 31) / 32 - k.begin / 32, 1);
    return k;
}

// What a workgroup keeps in LDS: o(w) is wave w's, of kFloats floats.
template <int D>
struct DecodeLds {
    static constexpr int kRow = D + 4;
    static constexpr int kFloats = 16 * kRow;
    float *o0, *o1, *o2, *o3;
    float (*m)[16];
    float (*l)[16];
    uint32_t* last;
    __device__ __forceinline__ float* o(int w) const { return w == 0 ? o0 : w == 1 ? o1 : w == 2 ? o2 : o3; }
};

// Workgroup wg of n_wg. EXACT: for a cap above kPlainCap (capped_tanh).
template <bool BF, int D, bool UNI, bool EXACT>
__device__ __forceinline__ void paged_decode(const PagedDecodeParams& p, uint32_t wg, uint32_t n_wg,
                                             const DecodeLds<D>& lds) {
    using Hf = Half16<BF>;
    constexpr int KS = D / 32, VEC = D / 16, VW = VEC / 2;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, g = lane >> 4, c = lane & 15;

    constexpr int kRow = DecodeLds<D>::kRow;
    float(*const s_m)[16] = lds.m;
    float(*const s_l)[16] = lds.l;

    // ---- the shares: running totals of the sequences' units, in every wave for
    // itself (no barrier): lane l holds sequences per * l .. + per - 1 ----
    const int per = (p.c.batch + 63) / 64;
    const uint32_t slabs = (uint32_t)(p.c.n_kv_heads * p.n_chunks);   // of one sequence
    const int b0 = min(lane * per, p.c.batch), b1 = min(b0 + per, p.c.batch);
    uint32_t steps = 0, mine = 0, longest = 0;
    int len0 = 0;   // the lane's last length (its only one where per is 1)
    for (int b = b0; b < b1; ++b) {
        len0 = p.c.lens[b];
        const uint32_t tiles = (uint32_t)keys_of(p, len0).tiles;
        longest = max(longest, tiles);
        steps += (tiles + kPdWaves - 1) / kPdWaves * slabs;
        mine += (tiles + kPieceUnits) * slabs;
    }
    // The work in units of a tile's time, cut into equal shares. Three ways, by the
    // longest slab and the number of tiles:
    //   each: there are no more slabs than workgroups, and not many fewer, and none is
    //         long: one slab each;
    //   few:  one workgroup per CU can do with one tile per wave: slabs are cut into
    //         such steps;
    //   else: the units are cut evenly, where a slab counts kPieceUnits more than its
    //         tiles, the time of its look-ups and its join.
    // GPU us: 64 sequences of 10 .. 300 tokens 11.9 cut evenly, 10.8 each; 32 ragged
    // ones 45.9, 33.4, 33.2 with 0, 2, 4 units; 256 of 10 .. 1000 tokens 130, 62.7, 55.7
    // (6: the same; 4 sequences of 500 .. 2000 tokens, 64 heads 12.5, 11.6 with 4, 6).
    uint32_t incl = wave_scan(steps);
    uint32_t total = lane_u32(incl, 63), share = kPdWaves, piece = 0;
    const uint32_t all_slabs = (uint32_t)p.c.batch * slabs;
    const bool each = all_slabs <= n_wg && all_slabs >= n_wg / 4 && !__any(longest > (uint32_t)kEachTiles);
    const bool few = !each && total <= (uint32_t)p.few_steps;
    if (each) {
        mine = (uint32_t)(b1 - b0) * slabs;
        incl = (uint32_t)b1 * slabs;
        total = all_slabs;
        share = 1;
    } else if (few) {
        mine = steps * kPdWaves;
        incl *= kPdWaves;
        total *= kPdWaves;
    } else {
        piece = kPieceUnits;
        incl = wave_scan(mine);
        total = lane_u32(incl, 63);
        share = max((total + n_wg - 1) / n_wg, 2u * kPdWaves);
    }
    auto cost_of = [&](int tiles) {
        return each ? 1u : few ? (uint32_t)(tiles + kPdWaves - 1) / kPdWaves * kPdWaves : (uint32_t)tiles + kPieceUnits;
    };
    uint32_t x = wg * share;
    const uint32_t x_end = min(x + share, total);

    while (x < x_end) {   // workgroup-uniform
        // ---- the sequence that unit x belongs to ----
        const int at_lane = __ffsll((unsigned long long)__ballot(incl > x)) - 1;
        uint32_t seq0 = lane_u32(incl - mine, at_lane);   // its first unit
        int b = at_lane, len = __builtin_amdgcn_readlane(len0, at_lane);
        if (per > 1) {
            b = at_lane * per;
            const int last_b = min(b + per, p.c.batch);
            for (;; b += 64) {   // ends: the lane's sequences hold unit x
                len = b + lane < last_b ? p.c.lens[b + lane] : 0;
                const uint32_t n = b + lane < last_b ? cost_of(keys_of(p, len).tiles) * slabs : 0u;
                const uint32_t upto = wave_scan(n);
                const uint64_t found = __ballot(seq0 + upto > x);
                if (found != 0 || b + 64 >= last_b) {
                    const int l = found != 0 ? __ffsll((unsigned long long)found) - 1 : 0;
                    seq0 += lane_u32(upto - n, l);
                    len = __builtin_amdgcn_readlane(len, l);
                    b += l;
                    break;
                }
                seq0 += lane_u32(upto, 63);
            }
        }
        b = __builtin_amdgcn_readfirstlane(b);
        const Keys keys = keys_of(p, len);
        const int tiles = __builtin_amdgcn_readfirstlane(keys.tiles);
        const int end = __builtin_amdgcn_readfirstlane(keys.end), begin = __builtin_amdgcn_readfirstlane(keys.begin);
        const uint32_t cost = cost_of(tiles);
        const uint32_t slab = __builtin_amdgcn_readfirstlane((x - seq0) / cost);
        const uint32_t unit0 = seq0 + slab * cost;   // its first unit
        // The piece: tiles [first, last) of the slab, whose tile t is its unit piece + t.
        // A slab of few tiles is not cut: it is its first unit's workgroup's.
        const bool uncut = each || tiles <= kUncutTiles;
        const int first = uncut ? 0 : max((int)(x - unit0) - (int)piece, 0);
        const int last = uncut ? tiles : min(max((int)(min(unit0 + cost, x_end) - unit0) - (int)piece, 0), tiles);
        const bool skip = uncut ? x != unit0 : first >= last;
        x = uncut ? unit0 + cost : min(unit0 + cost, x_end);
        if (skip) continue;
        int kvh = (int)slab, chunk = 0;
        if (p.n_chunks > 1) {
            kvh = (int)(slab / (uint32_t)p.n_chunks);
            chunk = (int)slab - kvh * p.n_chunks;
        }
        const int head0 = kvh * p.gqa + chunk * p.chunk_heads;
        const int nh = min(p.chunk_heads, p.gqa - chunk * p.chunk_heads);
        const int head = head0 + min(c, nh - 1);   // columns past the chunk repeat its last head
        const int pos = keys.len - 1;

        // This wave's tiles: base + 4 i, i < count.
        const int base = begin / 32 + first + wave;
        const int count = __builtin_amdgcn_readfirstlane((last - first - wave + kPdWaves - 1) / kPdWaves);
        const int* table_row = p.c.table + (long)b * p.c.max_pages;
        // Row offsets of 16 tiles ahead: lane l looks up octet l % 4 of the batch's tile l / 4.
        auto look_up = [&](int i0) {
            const int i = i0 + (lane >> 2);
            return octet_offset<D>(p.c, table_row, kvh, 32 * (base + kPdWaves * i) + 8 * (lane & 3), end);
        };
        long off, off_next;

        u32x4 qb[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            qb[ks] = load16(p.q + ((long)b * p.n_heads + head) * D + 32 * ks + 8 * g);
        const float slope = p.s.slopes ? p.s.slopes[head] * kLog2eF : 0.0f;

        f32x4 o[VEC];
        float m_run, l_run;   // of column c

        u32x4 kt[2][KS];
        uint32_t vt[8][VW];
        // Row offset of octet o of the batch's tile l0 / 4 (wave-uniform). An unmapped
        // octet reads the cache's first rows; its tokens are masked.
        auto octet_row = [&](int l0, int o) {
            const int lo = __builtin_amdgcn_readlane((int)(uint32_t)off, l0 + o);
            const int hi = __builtin_amdgcn_readlane((int)(off >> 32), l0 + o);
            return hi < 0 ? 0L : ((long)hi << 32) | (uint32_t)lo;
        };
        // Row offset for this lane, of octet 2 half + upper; with UNI the 32 tokens of a
        // tile share a page and octet 0's serves all.
        auto lane_row = [&](int l0, int half, int upper) {
            const long a = octet_row(l0, 2 * half), b2 = octet_row(l0, 2 * half + 1);
            return upper ? b2 : a;
        };
        auto load_k = [&](int i) {
            const int l0 = 4 * (i & 15);
            if constexpr (UNI) {
                const uint16_t* a = p.c.k + octet_row(l0, 0);
#pragma unroll
                for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
                        kt[blk][ks] = load16(a + (uint32_t)((16 * blk + c) * D + 32 * ks + 8 * g));
            } else {
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    const uint16_t* a = p.c.k + lane_row(l0, blk, c >> 3) + (c & 7) * D + 8 * g;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) kt[blk][ks] = load16(a + 32 * ks);
                }
            }
        };
        auto load_v1 = [&](uint32_t (&w)[VW], const uint16_t* a) {
            if constexpr (VEC == 8) {
                const u32x4 r = stream16(a);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = r[e];
            } else {
                const u32x2 r = stream8(a);
                w[0] = r[0];
                w[1] = r[1];
            }
        };
        auto load_v = [&](int i) {
            const int l0 = 4 * (i & 15);
            if constexpr (UNI) {
                const uint16_t* a = p.c.v + octet_row(l0, 0);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    load_v1(vt[e], a + (uint32_t)((16 * (e >> 2) + 4 * g + (e & 3)) * D + VEC * c));
            } else {
#pragma unroll
                for (int e2 = 0; e2 < 2; ++e2) {
                    const uint16_t* a = p.c.v + lane_row(l0, e2, g >> 1) + 4 * (g & 1) * D + VEC * c;
#pragma unroll
                    for (int e = 0; e < 4; ++e) load_v1(vt[4 * e2 + e], a + e * D);
                }
            }
        };

        // One pass over the tiles. An infinity in V must reach the rows that see it as one, but the
        // pair hi + lo makes NaN of it (lo may be zero or negative). So a piece whose sums hold NaN
        // where its weights do not is done again, with the values that are no numbers in a product
        // of their own, whose weights are 1. (Looking costs 0.1 .. 0.3 us a call, 1 .. 2 %.)
        auto pass = [&](auto careful) {
            constexpr bool kCareful = decltype(careful)::value;
            off = look_up(0);
            off_next = -1;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            m_run = kNoMax;
            l_run = 0.0f;   // (until the end: of this lane's tokens only)
            uint64_t unmapped = __ballot(off < 0);
            if (count > 0) {
                load_k(0);
                load_v(0);
            }
            if (count > 16) off_next = look_up(16);
            for (int i = 0; i < count; ++i) {
                const int t0 = 32 * (base + kPdWaves * i);
                const uint32_t gone = (uint32_t)(unmapped >> (4 * (i & 15))) & 15u;   // the tile's octets without a page
                float sc[8];
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) acc = Hf::mfma16(kt[blk][ks], qb[ks], acc);
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[4 * blk + r] = acc[r];
                }
                // K's registers are free: the next tile's keys are requested before this
                // tile's softmax, and its values (below) as soon as V's registers are.
                const bool more = i + 1 < count;
                if (more) {
                    if (((i + 1) & 15) == 0) {
                        off = off_next;
                        unmapped = __ballot(off < 0);
                        if (i + 17 < count) off_next = look_up(i + 17);
                    }
                    load_k(i + 1);
                }
                if constexpr (EXACT) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sc[e] = capped_tanh(sc[e], p.s) * p.s.cap_log2;
                } else if (p.s.cap_in != 0.0f) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sc[e] = capped(sc[e], p.s.cap_in, p.s.cap_log2);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sc[e] *= p.s.scale_log2;
                }
                const int tk = t0 + 4 * g;   // token of slot e: tk + 16 (e / 4) + e % 4
                if (p.s.slopes) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sc[e] = fmaf(-slope, (float)(pos - (tk + 16 * (e >> 2) + (e & 3))), sc[e]);
                }
                if (gone || t0 < begin || t0 + 32 > end) {   // wave-uniform
                    // Masked tokens: no score, and no value either (0 * NaN would stay NaN).
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int tok = tk + 16 * (e >> 2) + (e & 3);
                        const bool ok = tok >= begin && tok < end && !((gone >> (2 * (e >> 2) + (g >> 1))) & 1u);
                        if (!ok) {
                            sc[e] = -INFINITY;
#pragma unroll
                            for (int w = 0; w < VW; ++w) vt[e][w] = 0u;
                        }
                    }
                }
                float mx = sc[0];
#pragma unroll
                for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sc[e]);
                if (__any(mx > m_run)) {
                    mx = fmaxf(xor32_max(xor16_max(mx)), m_run);
                    const float a = kCareful ? join_weight(m_run - mx) : __builtin_amdgcn_exp2f(m_run - mx);
                    m_run = mx;
                    l_run *= a;
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[j][r] *= a;
                }
                const float sub = m_run - kPShift;
                u32x4 hi, lo;
                [[maybe_unused]] u32x4 seen;   // 1 for a token with a score
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(sc[e] - sub), p1 = __builtin_amdgcn_exp2f(sc[e + 1] - sub);
                    l_run += p0 + p1;
                    const uint32_t h2 = Hf::pack(p0, p1);
                    hi[e >> 1] = h2;
                    lo[e >> 1] = Hf::pack(p0 - Hf::to_f32((uint16_t)h2), p1 - Hf::to_f32((uint16_t)(h2 >> 16)));
                    if constexpr (kCareful) seen[e >> 1] = Hf::pack(sc[e] > -INFINITY, sc[e + 1] > -INFINITY);
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
                    u32x4 a;
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] = perm_b32(vt[2 * e + 1][j >> 1], vt[2 * e][j >> 1], sel);
                    if constexpr (kCareful) {
                        u32x4 bad;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            bad[e] = not_finite2<BF>(a[e]);
                            a[e] ^= bad[e];
                        }
                        o[j] = Hf::mfma16(bad, seen, o[j]);
                    }
                    o[j] = Hf::mfma16(a, hi, o[j]);
                    o[j] = Hf::mfma16(a, lo, o[j]);
                }
                if (more) load_v(i + 1);
            }
            l_run = xor32_sum(xor16_sum(l_run));
        };
        pass(std::false_type{});
        f32x4 all = o[0];   // NaN if any sum is (or where infinities of both signs are, which does no harm)
#pragma unroll
        for (int j = 1; j < VEC; ++j) all += o[j];
        const float any = (all[0] + all[1]) + (all[2] + all[3]);
        if (__any(any != any && l_run == l_run)) pass(std::true_type{});
        // ---- join the waves; write the output or hand the part over ----
        float* const mine_o = lds.o(wave);
        if (c < nh) {
            if (g == 0) {
                s_m[wave][c] = m_run;
                s_l[wave][c] = l_run;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < VEC; j += 4)
                    *reinterpret_cast<f32x4*>(mine_o + c * kRow + VEC * (4 * g + r) + j) =
                        f32x4{o[j][r], o[j + 1][r], o[j + 2][r], o[j + 3][r]};
        }
        __syncthreads();

        const int ch = VEC * (tid & 15);   // this thread's channels, of head tid / 16 (below, of h)
        float wm = kNoMax, wl = 0.0f, wo[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) wo[e] = 0.0f;
        // N parts (of which `live` count) into (wm, wl, wo).
        auto join = [&](auto n, int live, const float* m, const float* l, const float (*v)[VEC]) {
            constexpr int N = decltype(n)::value;
            float top = wm, w[N];
#pragma unroll
            for (int u = 0; u < N; ++u) {
                w[u] = u < live ? m[u] : kNoMax;
                top = fmaxf(top, w[u]);
            }
            const float a = join_weight(wm - top);
            wm = top;
            wl *= a;
#pragma unroll
            for (int e = 0; e < VEC; ++e) wo[e] *= a;
#pragma unroll
            for (int u = 0; u < N; ++u) {   // (the others' places hold anything)
                w[u] = join_weight(w[u] - top);
                wl = u < live ? fmaf(l[u], w[u], wl) : wl;
#pragma unroll
                for (int e = 0; e < VEC; ++e) wo[e] = u < live ? fmaf(v[u][e], w[u], wo[e]) : wo[e];
            }
        };
        auto join_lds = [&](int n, int h) {   // the first n <= 4 of the waves' places
            float m[kPdWaves], l[kPdWaves], v[kPdWaves][VEC];
#pragma unroll
            for (int w = 0; w < kPdWaves; ++w) {
                m[w] = s_m[w][h];
                l[w] = s_l[w][h];
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[w][e] = lds.o(w)[h * kRow + ch + e];
            }
            join(std::integral_constant<int, kPdWaves>{}, n, m, l, v);
        };
        if ((tid >> 4) < nh) join_lds(kPdWaves, tid >> 4);
        const bool whole = first == 0 && last == tiles;
        bool finish = whole;
        uint32_t wg0 = wg, wg1 = wg;   // the slab's workgroups
        const __amdgpu_buffer_rsrc_t ro =
            make_buffer_rsrc(p.part_o, (uint32_t)(2u * n_wg * p.chunk_heads * D * 4));
        if (!whole) {
            const uint32_t slot = 2u * wg + (first == 0 ? 1u : 0u);
            if ((tid >> 4) < nh) {
                const uint32_t row = slot * p.chunk_heads + (tid >> 4);
#pragma unroll
                for (int e = 0; e < VEC; e += 4)
                    publish_store16(ro, (row * D + ch + e) * 4u,
                                    make_u32x4(__float_as_uint(wo[e]), __float_as_uint(wo[e + 1]),
                                               __float_as_uint(wo[e + 2]), __float_as_uint(wo[e + 3])));
                if (ch == 0) {
                    publish_store(&p.part_ml[2 * row], wm);
                    publish_store(&p.part_ml[2 * row + 1], wl);
                }
            }
            if (first != 0) wg0 = (unit0 + piece) / share;
            if (last != tiles) wg1 = (unit0 + cost - 1) / share;
            publish_wait();
            __syncthreads();
            if (tid == 0) *lds.last = arrive_last(&p.counters[wg0], wg1 - wg0 + 1) ? 1u : 0u;
            __syncthreads();
            finish = *lds.last != 0;
            if (finish && tid == 0) p.counters[wg0] = 0u;   // zero for the next call
        }
        if (finish) {
            // The parts of the slab's workgroups. All threads fetch: groups of 16 threads per
            // head (rounded up to 4, 8 or 16 heads) take every groups-th part, eight of them
            // requested at a time (two where there are no more: each bypasses the L2, us,
            // one sequence of 700 tokens 8.7, 8.05), and are joined through LDS.
            const int span = nh <= 4 ? 4 : nh <= 8 ? 8 : 16;
            const int groups = 16 / span;
            const int h = (tid >> 4) & (span - 1);
            const int grp = __builtin_amdgcn_readfirstlane(tid / (16 * span));
            if (!whole) {
                const int parts = (int)(wg1 - wg0 + 1);
                const __amdgpu_buffer_rsrc_t rml =
                    make_buffer_rsrc(p.part_ml, (uint32_t)(2u * n_wg * p.chunk_heads * 2 * 4));
                wm = kNoMax;
                wl = 0.0f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) wo[e] = 0.0f;
                auto fetch = [&](auto batch, int i0) {   // parts i0, i0 + groups, ...
                    constexpr int N = decltype(batch)::value;
                    float m[N], l[N], v[N][VEC];
#pragma unroll
                    for (int u = 0; u < N; ++u) {
                        const int i = min(i0 + u * groups, parts - 1);
                        const uint32_t row = (2 * (wg0 + (uint32_t)i) + (i == 0 ? 1u : 0u)) * p.chunk_heads + h;
                        const u32x2 ml = publish_load8(rml, row * 8u);
                        const uint32_t mb = ml[0], lb = ml[1];
                        m[u] = __uint_as_float(mb);
                        l[u] = __uint_as_float(lb);
#pragma unroll
                        for (int e = 0; e < VEC; e += 4) {
                            const u32x4 r = publish_load16(ro, (row * D + ch + e) * 4u);
#pragma unroll
                            for (int e2 = 0; e2 < 4; ++e2) {
                                const uint32_t bits = r[e2];
                                v[u][e + e2] = __uint_as_float(bits);
                            }
                        }
                    }
                    join(batch, (parts - i0 + groups - 1) / groups, m, l, v);
                };
                if (h < nh) {
                    int i0 = grp;
                    for (; parts - i0 > 2 * groups; i0 += 8 * groups) fetch(std::integral_constant<int, 8>{}, i0);
                    if (i0 < parts) fetch(std::integral_constant<int, 2>{}, i0);
                }
            }
            if (groups > 1 && !whole) {   // workgroup-uniform
                __syncthreads();   // the waves' results are read
                if (h < nh) {
                    if (ch == 0) {
                        s_m[grp][h] = wm;
                        s_l[grp][h] = wl;
                    }
#pragma unroll
                    for (int e = 0; e < VEC; ++e) lds.o(grp)[h * kRow + ch + e] = wo[e];
                }
                __syncthreads();
                wm = kNoMax;
                wl = 0.0f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) wo[e] = 0.0f;
                if (h < nh && grp == 0) join_lds(groups, h);
            }
            if (h < nh && grp == 0 && p.own_o != nullptr) {
                const long at = (((long)kvh * p.c.batch + b) * p.gqa + chunk * p.chunk_heads + h + 1) * p.own_parts - 1;
#pragma unroll
                for (int e = 0; e < VEC; e += 4)
                    *reinterpret_cast<f32x4*>(p.own_o + at * D + ch + e) = f32x4{wo[e], wo[e + 1], wo[e + 2], wo[e + 3]};
                if (ch == 0) *reinterpret_cast<f32x2*>(p.own_ml + 2 * at) = f32x2{wm, wl};
            } else if (h < nh && grp == 0) {
                const float inv = wl > 0.0f || wl != wl ? 1.0f / wl : 0.0f;   // a row without keys is zero
                uint16_t* dst = p.out + ((long)b * p.n_heads + head0 + h) * D + ch;
                uint32_t w2[VW];
#pragma unroll
                for (int e = 0; e < VW; ++e) w2[e] = Hf::pack(wo[2 * e] * inv, wo[2 * e + 1] * inv);
                if constexpr (VEC == 8) *reinterpret_cast<u32x4*>(dst) = make_u32x4(w2[0], w2[1], w2[2], w2[3]);
                else *reinterpret_cast<u32x2*>(dst) = u32x2{w2[0], w2[1]};
            }
        }
        __syncthreads();   // the waves' results are read
    }
}

// ---------------------------------------------------------------- host

struct PagedDecodePlan {
    int workgroups, chunk_heads, n_chunks;
    size_t off_o, off_ml, bytes;
};

inline PagedDecodePlan plan_paged_decode(int batch, int n_heads, int n_kv_heads, int head_dim, long capacity, int cus) {
    PagedDecodePlan pl{};
    const int gqa = n_heads / n_kv_heads;
    pl.n_chunks = (gqa + 15) / 16;
    pl.chunk_heads = (gqa + pl.n_chunks - 1) / pl.n_chunks;
    const long slabs = (long)batch * n_kv_heads * pl.n_chunks;
    const long most = slabs * ((capacity + 31) / 32 / kPdWaves + 2);   // pieces of one tile per wave
    pl.workgroups = (int)std::max(1L, std::min((long)kPdPerCu * cus, most));
    const size_t slots = 2 * (size_t)pl.workgroups * pl.chunk_heads;
    pl.off_ml = kCounterBytes;
    pl.off_o = pl.off_ml + align_up(slots * 2 * sizeof(float), 256);
    pl.bytes = pl.off_o + align_up(slots * head_dim * sizeof(float), 256);
    return pl;
}

// The parameters of a call, over the workspace of its plan.
inline PagedDecodeParams paged_decode_params(const PagedLaunch& a, const PagedDecodePlan& pl) {
    PagedDecodeParams p{};
    p.q = static_cast<const uint16_t*>(a.q);
    p.out = static_cast<uint16_t*>(a.out);
    p.c = paged_view(a);
    p.s = score_opts(a);
    p.n_heads = a.n_heads;
    p.gqa = a.n_heads / a.n_kv_heads;
    p.n_chunks = pl.n_chunks;
    p.chunk_heads = pl.chunk_heads;
    char* ws = static_cast<char*>(a.workspace);
    p.counters = reinterpret_cast<uint32_t*>(ws);
    p.part_ml = reinterpret_cast<float*>(ws + pl.off_ml);
    p.part_o = reinterpret_cast<float*>(ws + pl.off_o);
    p.few_steps = std::min(device_cu_count(), pl.workgroups);
    return p;
}

}  // namespace llmik
