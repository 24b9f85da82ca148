// Attention of many query rows over a paged cache: prompts (ragged chunks of new
// tokens, causal by position) and the shared prefix of a decoding batch.
//
// Rows. All query rows that read one KV head's keys form one list: row r of a
// sequence is query token r / G, head r % G of the KV head's G query heads (for
// the prefix: sequence r / G of the batch). A workgroup takes 128 consecutive
// rows, 32 per wave, so that short chunks of several heads fill a tile as long
// prompts do, and walks the keys in 64-token tiles.
//
// Products on 32x32x16 matrix instructions, transposed so that a lane keeps one
// row's softmax:
//   S^T = K Q^T: A = 32 keys from LDS, B = the wave's 32 rows (registers): lane
//     (h, n) gets row n's scores of tokens 8 i + 4 h + 0..3, i < 4;
//   O^T = V^T P^T: the scores are the B operand as they lie (k-slots 8h .. 8h + 7
//     of a 16-token step are its tokens 4h .. + 3 and 8 + 4h .. + 3); A is V read
//     from LDS by the transposing 64-bit read (16 lanes give four tokens' 16
//     channels and get one channel's four tokens each).
// P is rounded once to 16 bits, as 2^8 p (fp16 keeps its full precision down to
// 2^-22); sums and statistics are fp32.
//
// K and V tiles are copied to LDS asynchronously, one tile ahead. The 16-byte
// chunks of a row are permuted (xor with the row number) so that the operand
// reads of eight rows fall into different banks; the copies place them so.
//
// Where there are fewer row tiles than two workgroups per CU, their keys are cut into
// parts, whose sums a second kernel joins (paged_flash.hip, paged_prefix.hip).
//
// Measured: a prompt of 8192 tokens, 32 heads over 8 KV heads of 128, bf16: 518 .. 570
// us, 0.96 .. 1.06 PFLOP/s (a large matrix product reaches 1.42): the matrix units work 57 % of
// the cycles and vector instructions (4.7 a score, the products not counted) about half of
// them, which overlap little. Of 2048 tokens 50 .. 56 us, twice the products' time: a CU's
// longer workgroup ends alone, one wave per SIMD. Of 2000 tokens with heads of 64 35 us: the
// vector work of heads of 128 on half of the products. Chunks of four prompts over up to
// 6000 cached tokens, capped scores: 161 .. 175 us, 0.67 .. 0.72 PFLOP/s, bound by the cap's
// two transcendentals per score. Three short prompts 8.2 us: launch, look-ups, two or three
// tiles (12.8 with a table for 1024 tokens or more, where plan_prefill cuts keys and launches
// the join).
#pragma once

#include "paged_common.hpp"

namespace llmik {

constexpr int kPfThreads = 256;
constexpr int kPfRows = 128;    // query rows of a workgroup
constexpr int kPfTileLog = 6;   // tokens of a tile
constexpr int kPfTile = 1 << kPfTileLog;
constexpr float kPLag = 6.0f;     // by so much (log2) may a score pass the exponents' reference

struct PagedFlashParams {
    const uint16_t* q;
    uint16_t* out;
    PagedView c;
    ScoreOpts s;
    const int* cu;            // [batch + 1]
    int rows;                 // rows of q
    uint32_t per_round;       // workgroups of one per CU
    int n_heads;
    FastDiv gqa;
    int base;                 // the ragged form: workgroups without parts
    int splits;               // parts of a tile's keys at most (the prefix form: exactly)
    float* part_o;            // ragged: [tiles * n_kv_heads, splits, kPfRows, D] and (m, l); prefix: [n_kv_heads,
    float* part_ml;           //   rows, splits + 1, D] and (m, l), the last one not this kernel's
    const int* prefix_pages;  // the prefix form
    int prefix_len, chunk;
};

// A workgroup's 128 rows: row tile `tile` of sequence b, whose `rows` query tokens
// begin at row row0 of q and at position pos0. (The prefix form: row i is sequence i.)
struct RowTile {
    int b, tile, row0, rows, pos0;
};

__device__ __forceinline__ int oldest_key(const ScoreOpts& s, int pos) {   // of those that a query at pos sees
    return pos >= s.window ? pos - s.window + 1 : 0;
}

// Row tile number `item` of the call, false past the last (the grid is an upper
// bound). Every wave counts the sequences' tiles for itself: lane l holds sequences
// per * l .. + per - 1.
__device__ __forceinline__ bool find_tile(const PagedFlashParams& p, uint32_t item, RowTile& t) {
    const int lane = threadIdx.x & 63;
    const int per = (p.c.batch + 63) / 64;
    const int b0 = min(lane * per, p.c.batch), b1 = min(b0 + per, p.c.batch);
    auto tokens_of = [&](int b, int& row0) {   // query tokens of sequence b, kept inside q
        row0 = max(p.cu[b], 0);
        return max(min(p.cu[b + 1], p.rows) - row0, 0);
    };
    auto tiles_of = [&](int b) {
        int row0;
        return (uint32_t)(tokens_of(b, row0) * (int)p.gqa.d + kPfRows - 1) / kPfRows;
    };
    uint32_t mine = 0;
    int row0 = 0, rows = 0, pos0 = 0;   // the lane's only sequence, where per is 1: one round trip less
    if (per == 1 && b0 < b1) {
        const int len = max(p.c.lens[b0], 0), stop = p.cu[b0 + 1];
        rows = tokens_of(b0, row0);
        mine = (uint32_t)(rows * (int)p.gqa.d + kPfRows - 1) / kPfRows;
        pos0 = len - (stop - row0);
    } else {
        for (int b = b0; b < b1; ++b) mine += tiles_of(b);
    }
    const uint32_t incl = wave_scan(mine);
    const uint32_t total = lane_u32(incl, 63);
    if (item >= total) return false;
    // The call's last tiles come first: of one prompt those that see the most keys.
    // (Between sequences the order is the batch's, whatever their lengths.) Where all
    // workgroups run at once, two per CU, the second half goes the other way, so that a
    // CU's two have about the same work together as another's. (Of heads of 64 three fit a
    // CU; the rule counts two.)
    const uint32_t half = p.per_round / (uint32_t)(p.c.n_kv_heads * p.splits);   // tiles of one workgroup per CU
    uint32_t x = total - 1 - item;
    if (item >= half && total <= 2 * half) x = item - half;
    const int at_lane = __ffsll((unsigned long long)__ballot(incl > x)) - 1;
    uint32_t first = lane_u32(incl - mine, at_lane);   // the sequence's first tile
    int b = at_lane;
    if (per > 1) {
        b = at_lane * per;
        const int last_b = min(b + per, p.c.batch);
        for (;; b += 64) {   // ends: the lane's sequences hold tile x
            const uint32_t n = b + lane < last_b ? tiles_of(b + lane) : 0u;
            const uint32_t upto = wave_scan(n);
            const uint64_t found = __ballot(first + upto > x);
            if (found != 0 || b + 64 >= last_b) {
                const int l = found != 0 ? __ffsll((unsigned long long)found) - 1 : 0;
                first += lane_u32(upto - n, l);
                b += l;
                break;
            }
            first += lane_u32(upto, 63);
        }
    }
    t.b = __builtin_amdgcn_readfirstlane(b);
    t.tile = __builtin_amdgcn_readfirstlane((int)(x - first));
    if (per == 1) {
        t.rows = __builtin_amdgcn_readlane(rows, t.b);
        t.row0 = __builtin_amdgcn_readlane(row0, t.b);
        t.pos0 = __builtin_amdgcn_readlane(pos0, t.b);
    } else {
        t.rows = __builtin_amdgcn_readfirstlane(tokens_of(t.b, t.row0));
        t.row0 = __builtin_amdgcn_readfirstlane(t.row0);
        t.pos0 = __builtin_amdgcn_readfirstlane(max(p.c.lens[t.b], 0) - (p.cu[t.b + 1] - t.row0));
    }
    return true;
}

// The keys [begin, end) that a row tile's rows see, in `tiles` tiles of 64 tokens, and
// the parts (of part_tiles tiles) that they are cut into (parts_of, p.splits at most).
constexpr int kMaxParts = 8;
constexpr int kMinPart = 4;   // tiles of a part at least

// The number of parts for `tiles` key tiles where the call has `base` workgroups uncut,
// from heads of 128 (those of 64 have half the sums and less than half of a tile's time).
// A tile takes 1.3 us, a part's sums (64 KiB) are written and read again: per workgroup
// and part 0.026 us of the card's time. tiles * 1.3 / n + base * 0.026 * n is least at
// n^2 = 50 tiles / base (here the nearest n). Measured with n = 1, 2, 3, 4, 5, 6, 8: two sequences of 100 rows
// over up to 1214 tokens (base 40) 28.6, 21.9, 17.9, 16.5, 15.7, 15.9, 15.2; three of up
// to 199 over up to 2271 (base 80) 48.9, 34.0, 28.4, 24.9, 24.2, 27.2, 27.4; 400 over 244
// (base 104) 18.3, 19.2, 19.8, 20.5, 20.8, 21.1, 21.8 (the join's launch, 3 us, included).
__host__ __device__ __forceinline__ int parts_of(uint32_t tiles, uint32_t base) {   // tiles <= 2^24, base <= 2^24
    uint32_t n = 1;
#pragma unroll
    for (uint32_t k = 2; k <= kMaxParts; ++k)
        n = (2 * k - 1) * (2 * k - 1) * base <= 200 * tiles && k * kMinPart <= tiles ? k : n;
    return (int)n;
}
struct TileKeys {
    int lo, hi;   // positions of the first and the last row
    int begin, end, tiles, parts, part_tiles;
};
__device__ __forceinline__ TileKeys keys_of_tile(const PagedFlashParams& p, const RowTile& t) {
    const int n_rows = t.rows * (int)p.gqa.d, r0 = t.tile * kPfRows;
    TileKeys k;
    k.lo = t.pos0 + (int)p.gqa.div((uint32_t)r0);
    k.hi = t.pos0 + (int)p.gqa.div((uint32_t)min(r0 + kPfRows, n_rows) - 1u);
    k.begin = oldest_key(p.s, k.lo) / kPfTile * kPfTile;
    k.end = min(p.c.capacity, k.hi + 1);
    k.tiles = k.end > k.begin ? (k.end - k.begin + kPfTile - 1) / kPfTile : 0;
    k.parts = p.splits > 1 ? min(p.splits, parts_of((uint32_t)k.tiles, (uint32_t)p.base)) : 1;
    k.part_tiles = (k.tiles + k.parts - 1) / k.parts;
    if (k.parts > 1) k.parts = (k.tiles + k.part_tiles - 1) / k.part_tiles;
    return k;
}

// What a workgroup keeps in LDS: two tiles of K and of V. (Separate arrays: the
// compiler then knows that a tile's copies and the other's reads are apart.)
template <int D>
struct FlashLds {
    static constexpr int kTileBytes = kPfTile * D * 2;
    uint8_t *k0, *k1, *v0, *v1;
    int *lo, *hi;              // [4]
    uint32_t* bad;             // some V is no number (see the end of paged_flash)
};

// Workgroup wg of n_wg. EXACT: for a cap above kPlainCap (capped_tanh; a kernel of its
// own, as its instructions beside the others cost all calls: us, 8192 tokens 565, 583
// with it, 2048 tokens 52.9, 55.5. Four chunks over up to 6000 tokens with a cap of 50
// 167, of 1000 202).
template <bool BF, int D, bool PREFIX, bool EXACT>
__device__ __forceinline__ void paged_flash(const PagedFlashParams& p, uint32_t wg, uint32_t n_wg,
                                            const FlashLds<D>& lds) {
    using Hf = Half16<BF>;
    constexpr int KS = D / 16, CB = D / 32;
    constexpr int CPR = D / 8;                    // 16-byte chunks of a row
    constexpr int kRowBytes = D * 2;
    constexpr int kCopies = 16 * CPR / 64;        // copy instructions for a wave's 16 rows
    constexpr int kRowsPerCopy = 64 / CPR;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, h = lane >> 5, n = lane & 31;

    uint8_t *const s_k0 = lds.k0, *const s_k1 = lds.k1, *const s_v0 = lds.v0, *const s_v1 = lds.v1;
    int *const s_lo = lds.lo, *const s_hi = lds.hi;
    uint32_t& s_bad = *lds.bad;

    const int kvh = (int)(wg % (uint32_t)p.c.n_kv_heads);
    const uint32_t item = wg / (uint32_t)(p.c.n_kv_heads * p.splits);
    const int split = (int)(wg / (uint32_t)p.c.n_kv_heads % (uint32_t)p.splits);
    const int G = (int)p.gqa.d;

    // ---- the workgroup's rows ----
    RowTile ft{};
    if constexpr (PREFIX) {
        ft.tile = (int)item;
        ft.rows = p.c.batch;
    } else {
        const int used = p.cu[p.c.batch];
        const bool found = find_tile(p, item, ft);
        // Rows that belong to no sequence (a padded batch) are zeroed, by all workgroups together.
        const long chunks = (long)p.n_heads * CPR;
        const long at0 = (long)wg * kPfThreads + tid, step = (long)n_wg * kPfThreads;
        for (long i = min(max(used, 0), p.rows) * chunks + at0; i < p.rows * chunks; i += step)
            *reinterpret_cast<u32x4*>(p.out + 8 * i) = u32x4{0u, 0u, 0u, 0u};
        if (!found) return;
    }
    const int n_rows = ft.rows * G;
    const int r_wave = ft.tile * kPfRows + 32 * wave;   // the wave's first row
    const bool live = r_wave < n_rows;                  // wave-uniform
    const int r = min(r_wave + n, n_rows - 1);          // rows past the end repeat the last
    const int qi = (int)p.gqa.div((uint32_t)r);
    const int head = kvh * G + (r - qi * G);
    const long q_row = (PREFIX ? (long)qi : (long)ft.row0 + qi) * p.n_heads + head;
    const int pos = PREFIX ? max(p.c.lens[qi], 0) - 1 : ft.pos0 + qi;
    // ---- the keys that any of them sees, [begin, end), in 64-token tiles ----
    auto oldest = [&](int at) { return oldest_key(p.s, at); };
    int begin, end, tiles, parts = 1;
    int pos_lo, pos_hi, wg_lo, wg_hi;   // positions of the wave's rows, of the workgroup's
    if constexpr (PREFIX) {
        pos_lo = pos_hi = pos;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            pos_lo = min(pos_lo, __shfl_xor(pos_lo, d));
            pos_hi = max(pos_hi, __shfl_xor(pos_hi, d));
        }
        if (lane == 0) {
            s_lo[wave] = live ? pos_lo : INT_MAX;
            s_hi[wave] = live ? pos_hi : -1;
        }
        __syncthreads();
        wg_lo = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3]));
        wg_hi = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3]));
        begin = max(split * p.chunk, oldest(wg_lo)) / kPfTile * kPfTile;
        end = min(min(split * p.chunk + p.chunk, p.prefix_len), wg_hi + 1);
        tiles = end > begin ? (end - begin + kPfTile - 1) / kPfTile : 0;
    } else {
        pos_lo = ft.pos0 + (int)p.gqa.div((uint32_t)min(r_wave, n_rows - 1));
        pos_hi = ft.pos0 + (int)p.gqa.div((uint32_t)min(r_wave + 31, n_rows - 1));
        const TileKeys k = keys_of_tile(p, ft);
        wg_lo = k.lo;
        wg_hi = k.hi;
        parts = k.parts;
        if (split >= parts) return;
        begin = k.begin + split * k.part_tiles * kPfTile;
        end = min(k.end, begin + k.part_tiles * kPfTile);
        tiles = min(k.part_tiles, k.tiles - split * k.part_tiles);
    }
    if (tiles <= 0) tiles = begin = end = 0;
    pos_lo = __builtin_amdgcn_readfirstlane(pos_lo);
    pos_hi = __builtin_amdgcn_readfirstlane(pos_hi);
    wg_lo = __builtin_amdgcn_readfirstlane(wg_lo);
    wg_hi = __builtin_amdgcn_readfirstlane(wg_hi);
    begin = __builtin_amdgcn_readfirstlane(begin);
    end = __builtin_amdgcn_readfirstlane(end);
    tiles = __builtin_amdgcn_readfirstlane(tiles);

    // Tiles that all of the wave's rows see wholly, that some row sees, and that all rows
    // of the workgroup see wholly: [lo, hi).
    const int full_lo = (oldest(pos_hi) - begin + kPfTile - 1) >> kPfTileLog;
    const int full_hi = (min(end, pos_lo + 1) - begin) >> kPfTileLog;
    const int seen_lo = (oldest(pos_lo) - begin) >> kPfTileLog;
    const int seen_hi = live ? ((pos_hi - begin) >> kPfTileLog) + 1 : INT_MIN;
    const int wg_full_lo = (oldest(wg_hi) - begin + kPfTile - 1) >> kPfTileLog;
    const int wg_full_hi = (wg_lo + 1 - begin) >> kPfTileLog;

    // ---- copies: wave w brings tokens 16 w .. + 15 of every tile ----
    // Every wave looks up all octets, eight tiles at a time: lane l octet l % 8 of tile
    // i0 + l / 8. A copy is a load from a buffer of the octet's rows in front of the end;
    // rows behind it, or without a page, lie outside the buffer's range and come as
    // zeros (their scores are masked, and their values must not turn 0 * v into NaN).
    const int* table_row = PREFIX ? p.prefix_pages : p.c.table + (long)ft.b * p.c.max_pages;
    auto token_of = [&](int i0) { return begin + kPfTile * (i0 + (lane >> 3)) + 8 * (lane & 7); };
    auto look_up = [&](int i0) { return octet_offset<D>(p.c, table_row, kvh, token_of(i0), end); };
    int at_lo, at_hi, at_bytes;   // the lane's octet of the batch: its place in bytes, its rows' bytes
    uint64_t batch_gone;          // lanes whose octet has no page (or lies behind the end)
    auto adopt = [&](long off, int i0) {
        const bool gone = off < 0;
        const long at = gone ? 0L : 2 * off;
        at_lo = (int)(uint32_t)at;
        at_hi = (int)(at >> 32);
        at_bytes = gone ? 0 : min(max(end - token_of(i0), 0), 8) * kRowBytes;
        batch_gone = __ballot(gone);
    };
    const long off_first = look_up(0);
    u32x4 qb[KS];   // (requested behind the look-up, which is waited for first)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qb[ks] = load16(p.q + q_row * D + 16 * ks + 8 * h);
    const float slope = p.s.slopes ? p.s.slopes[head] * kLog2eF : 0.0f;
    adopt(off_first, 0);
    long off_next = tiles > 8 ? look_up(8) : -1L;
    // Copy instruction c fills rows kRowsPerCopy c .. of the wave's 16: lane l writes
    // chunk slot l % CPR of row l / CPR, i.e. the chunk that the permutation puts there.
    const int crow = lane / CPR, cslot = lane % CPR;
    __amdgpu_buffer_rsrc_t rk[2], rv[2];   // of the wave's two octets of the tile being copied
    uint32_t gone_next = 0;                // bit o: octet o of that tile has no page
    // (Where there is no tile i nothing is read.)
    auto prepare = [&](int i) {
        if ((i & 7) == 0 && i) {
            adopt(off_next, i);
            off_next = i + 8 < tiles ? look_up(i + 8) : -1L;
        }
        const int l0 = 8 * (i & 7);
        gone_next = (uint32_t)(batch_gone >> l0) & 255u;
#pragma unroll
        for (int o8 = 0; o8 < 2; ++o8) {
            const int l = l0 + 2 * wave + o8;
            const long at = ((long)__builtin_amdgcn_readlane(at_hi, l) << 32) |
                            (uint32_t)__builtin_amdgcn_readlane(at_lo, l);
            const uint32_t bytes = (uint32_t)__builtin_amdgcn_readlane(at_bytes, l);
            rk[o8] = make_buffer_rsrc(reinterpret_cast<const uint8_t*>(p.c.k) + at, bytes);
            rv[o8] = make_buffer_rsrc(reinterpret_cast<const uint8_t*>(p.c.v) + at, bytes);
        }
    };
    auto copy = [&](uint8_t* dst, bool is_v, int c) {
        const int row = kRowsPerCopy * c + crow, trow = 16 * wave + row;   // of the wave's 16, of the tile
        const int chunk = cslot ^ (is_v ? (D == 128 ? (trow & 3) << 2 : ((trow >> 1) & 1) << 2)
                                        : (D == 128 ? trow & 15 : trow & 7));
        const int octet = (kRowsPerCopy * c) / 8;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            is_v ? rv[octet] : rk[octet],
            (__attribute__((address_space(3))) void*)(dst + (16 * wave + kRowsPerCopy * c) * kRowBytes), 16,
            (row & 7) * kRowBytes + 16 * chunk, 0, 0, 0);
    };

    f32x16 o[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[cb][e] = 0.0f;
    float m_run = kNoMax, l_run = 0.0f;   // of row n; l_run: this lane's tokens only
    // sc * mult + add are the scores in the log2 domain: sc as it comes from the products,
    // or -1 / (e^2x + 1) where there is a cap (the rest of cap * tanh x is mult and add; with
    // EXACT tanh x), or, with a bias or a negative scale, the score itself (mult must be
    // positive: the masked value, -inf, must stay the smallest).
    const bool cap = p.s.cap_in != 0.0f, modified = p.s.slopes != nullptr || (!cap && p.s.scale_log2 <= 0.0f);
    const float mult = modified ? 1.0f : EXACT ? p.s.cap_log2 : cap ? 2.0f * p.s.cap_log2 : p.s.scale_log2;
    const float add = cap && !modified && !EXACT ? p.s.cap_log2 : 0.0f;

    // LDS offsets of this lane's operand reads.
    const uint32_t k_row = (uint32_t)(n * kRowBytes);
    const uint32_t k_sw = (uint32_t)((h ^ (D == 128 ? n & 15 : n & 7)) * 16);
    const int vr = (lane & 15) >> 2;                        // token of the group's four
    const uint32_t v_chunk = (uint32_t)(2 * ((lane >> 4) & 1) + ((lane & 3) >> 1));
    const uint32_t v_sw = (uint32_t)(D == 128 ? vr << 2 : (vr >> 1) << 2);
    const uint32_t v_at = (uint32_t)((4 * h + vr) * kRowBytes) + 8 * (lane & 1);

    // copies(0, c), copies(1, c): copy c of the next tile's K and of its V, issued among
    // the products of the two blocks' scores, whose time hides them: before all work they
    // waited for the CU's one vector memory path, 1000 of a tile's 3900 cycles (us, a
    // prompt of 8192 tokens 562 -> 550, 2048 tokens 58.2 -> 54.5, chunks 198 -> 189;
    // spread further down to the products with V they come too late: 542, 56.9, 210).
    auto compute = [&](const uint8_t* sk, const uint8_t* sv, int i, uint32_t gone, auto copies) {
        const int t0 = begin + kPfTile * i;
        float sc[32];
        // K's operands are requested eight products ahead, in this order: left to itself the
        // compiler saves the registers and waits for each (us, 8192 tokens 562 -> 536,
        // 2048 tokens 56.9 -> 52.5, chunks 195 -> 180).
        u32x4 ka[2][KS];
        auto load_k = [&](int blk, int ks) {
            ka[blk][ks] = *reinterpret_cast<const u32x4*>(sk + k_row + 32 * blk * kRowBytes + (k_sw ^ (32u * ks)));
        };
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) load_k(0, ks);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            f32x16 acc;
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                acc = Hf::mfma32(ka[blk][ks], qb[ks], acc);
                if (blk == 0) load_k(1, ks);
                if (ks % 2 == 1) copies(blk, ks / 2);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[16 * blk + e] = acc[e];
        }
        // value e belongs to token t0 + 4 h + 8 (e / 4) + e % 4
        const int tk = t0 + 4 * h;
        if constexpr (EXACT) {
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < 32; ++e) top = fmaxf(top, fabsf(sc[e]));
            if (__any(top * fabsf(p.s.cap_x) >= 0.5f)) {
#pragma unroll
                for (int e = 0; e < 32; ++e) sc[e] = capped_tanh(sc[e], p.s);
            } else {   // what scores are below a cap that is far from most
#pragma unroll
                for (int e = 0; e < 32; ++e) sc[e] = tanh_series(sc[e] * p.s.cap_x);
            }
        } else if (cap) {
#pragma unroll
            for (int e = 0; e < 32; ++e) sc[e] = capped_part(sc[e], p.s.cap_in);
        }
        if (modified) {
            const float by = EXACT ? p.s.cap_log2 : cap ? 2.0f * p.s.cap_log2 : p.s.scale_log2;
            const float plus = cap && !EXACT ? p.s.cap_log2 : 0.0f;
#pragma unroll
            for (int e = 0; e < 32; ++e) sc[e] = fmaf(sc[e], by, plus);
            if (p.s.slopes) {
#pragma unroll
                for (int e = 0; e < 32; ++e) sc[e] = fmaf(-slope, (float)(pos - (tk + 8 * (e >> 2) + (e & 3))), sc[e]);
            }
        }
        if (gone || i < full_lo || i >= full_hi) {   // wave-uniform
            const int old = oldest(pos), lim = min(pos + 1, end);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const int tok = tk + 8 * (e >> 2) + (e & 3);
                if (tok < old || tok >= lim || ((gone >> (e >> 2)) & 1u)) sc[e] = -INFINITY;
            }
        }
        // Exponents (of 2^kPShift p) against the reference m_run, which is moved only
        // when a score passes it by kPLag: 2^kPShift p stays below 2^(kPShift + kPLag),
        // and most tiles rescale nothing.
        float t[32], mx = -INFINITY;
        const float sub = m_run - kPShift;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            t[e] = fmaf(sc[e], mult, add - sub);
            mx = fmaxf(mx, t[e]);
        }
        if (__any(mx > kPShift + kPLag)) {
            mx = fmaxf(xor32_max(mx), kPShift);
            float m_new = sub + mx;
            if (m_run == kNoMax) {   // the first keys: the scores themselves (m_run + mx has none of their bits)
                m_new = -INFINITY;
#pragma unroll
                for (int e = 0; e < 32; ++e) m_new = fmaxf(m_new, fmaf(sc[e], mult, add));
                m_new = fmaxf(xor32_max(m_new), kNoMax);
            }
            const float a = join_weight(m_run - m_new);
            m_run = m_new;
            l_run *= a;
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[cb][e] *= a;
#pragma unroll
            for (int e = 0; e < 32; ++e) t[e] = fmaf(sc[e], mult, add + (kPShift - m_run));
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) t[e] = __builtin_amdgcn_exp2f(t[e]);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            u32x4 pb;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t p2 = Hf::pack(t[8 * kk + 2 * e], t[8 * kk + 2 * e + 1]);
                pb[e] = p2;
                l_run = Hf::add_pair(p2, l_run);   // the sum of what the products use
            }
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                const uint8_t* a = sv + v_at + 16 * kk * kRowBytes + 16 * ((v_chunk + 4 * cb) ^ v_sw);
                typedef short s16x4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a);
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a + 8 * kRowBytes));
                const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
                o[cb] = Hf::mfma32(make_u32x4(l2[0], l2[1], h2[0], h2[1]), pb, o[cb]);
            }
        }
    };

    // One tile ahead: a tile's copies are complete for the whole workgroup, and the
    // other buffer is read, once every wave has waited for its own copies and
    // passed the barrier.
    auto turn = [&](uint8_t* k_cur, uint8_t* v_cur, uint8_t* k_far, uint8_t* v_far, int i) {
        __builtin_amdgcn_s_waitcnt(0);
        asm volatile("s_barrier" ::: "memory");
        const uint32_t gone = gone_next;
        prepare(i + 1);
        auto copies = [&](int v, int c) { copy(v ? v_far : k_far, v, c); };
        // Where some row does not see some token, every wave looks through its 16 rows of V
        // for infinities and NaN (bits of |x| from the type's infinity on): a probability
        // of 0 would make NaN of them. Such a tile's rows are done again, below.
        if (i < wg_full_lo || i >= wg_full_hi) {   // workgroup-uniform
            u32x4 w[kCopies];
#pragma unroll
            for (int c = 0; c < kCopies; ++c)
                w[c] = *reinterpret_cast<const u32x4*>(v_cur + 16 * wave * kRowBytes + 1024 * c + 16 * lane);
            __builtin_amdgcn_sched_barrier(0);   // (one wait for all)
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < kCopies; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = w[c][e];
                    top = max_abs2(top, x);
                }
            const uint32_t inf = BF ? 0x7F80u : 0x7C00u;
            if ((top & 0xFFFFu) >= inf || (top >> 16) >= inf) s_bad = 1u;
        }
        if (i >= seen_lo && i < seen_hi) {
            compute(k_cur, v_cur, i, gone, copies);
        } else {   // no row of this wave sees a key of it
#pragma unroll
            for (int c = 0; c < 2 * kCopies; ++c) copies(c / kCopies, c % kCopies);
        }
    };
    if (tid == 0) s_bad = 0u;   // (the first turn's barrier follows)
    if (tiles > 0) {
        prepare(0);
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
            copy(s_k0, false, c);
            copy(s_v0, true, c);
        }
    }
    for (int i = 0; i < tiles; i += 2) {
        turn(s_k0, s_v0, s_k1, s_v1, i);
        if (i + 1 < tiles) turn(s_k1, s_v1, s_k0, s_v0, i + 1);
    }
    __builtin_amdgcn_s_waitcnt(0);   // no copy into LDS outlives the workgroup

    l_run = xor32_sum(l_run);
    // The row's place among the parts.
    auto part_at = [&](int row) {
        return PREFIX ? ((long)kvh * n_rows + ft.tile * kPfRows + row) * (p.splits + 1) + split
                      : (((long)item * p.c.n_kv_heads + kvh) * p.splits + split) * kPfRows + row;
    };
    const bool as_part = PREFIX || parts > 1;
    // The wave's rows go through LDS, so that whole rows are stored, 16 bytes a lane: from
    // the registers a store of outputs has 64 pieces of 8 bytes, a row apart (us, three
    // short prompts 8.96, 8.15 through LDS), one of parts pieces of 16, which wins where
    // few rows are there (64 sequences behind 8192 tokens 31.1, 29.7 through LDS, 6 behind
    // 1500 10.3, 10.9). Chunks of 16 bytes are permuted like the tiles'.
    const bool direct = as_part && ft.tile * kPfRows + kPfRows > n_rows;
    const int n_live = min(n_rows - r_wave, 32);   // rows of the wave; none: <= 0
    uint8_t* const rows_at = wave == 0 ? s_k0 : wave == 1 ? s_k1 : wave == 2 ? s_v0 : s_v1;
    auto place = [&](int row, int chunk, int chunks) {
        return rows_at + 16 * (row * chunks + (chunk ^ (row & (chunks - 1))));
    };
    auto quad = [&](int cb, int e) { return f32x4{o[cb][e], o[cb][e + 1], o[cb][e + 2], o[cb][e + 3]}; };
    __syncthreads();   // the tiles are read
    if (live && as_part) {
        constexpr int kChunks = D / 4;
        const long at = part_at(32 * wave + n);
        if (h == 0 && n < n_live) *reinterpret_cast<f32x2*>(p.part_ml + 2 * at) = f32x2{m_run, l_run};
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int c = 8 * cb + e / 2 + h;
                if (!direct) *reinterpret_cast<f32x4*>(place(n, c, kChunks)) = quad(cb, e);
                else if (n < n_live) *reinterpret_cast<f32x4*>(p.part_o + at * D + 4 * c) = quad(cb, e);
            }
        if (!direct) {
#pragma unroll
            for (int j = 0; j < kChunks / 2; ++j) {
                const int row = (64 * j + lane) / kChunks, c = lane % kChunks;
                const u32x4 v = *reinterpret_cast<const u32x4*>(place(row, c, kChunks));
                *reinterpret_cast<u32x4*>(p.part_o + part_at(32 * wave + row) * D + 4 * c) = v;   // (all rows live)
            }
        }
    } else if (live) {
        constexpr int kChunks = D / 8;
        const float inv = l_run > 0.0f || l_run != l_run ? 1.0f / l_run : 0.0f;   // a row without keys is zero
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const f32x4 v = quad(cb, e);
                *reinterpret_cast<u32x2*>(place(n, 4 * cb + e / 4, kChunks) + 8 * h) =
                    u32x2{Hf::pack(v[0] * inv, v[1] * inv), Hf::pack(v[2] * inv, v[3] * inv)};
            }
#pragma unroll
        for (int j = 0; j < kChunks / 2; ++j) {
            const int row = (64 * j + lane) / kChunks, c = lane % kChunks, rw = r_wave + row;
            const u32x4 v = *reinterpret_cast<const u32x4*>(place(row, c, kChunks));
            const int qr = (int)p.gqa.div((uint32_t)rw);
            const long to = ((long)ft.row0 + qr) * p.n_heads + kvh * G + (rw - qr * G);
            if (row < n_live) *reinterpret_cast<u32x4*>(p.out + to * D + 8 * c) = v;
        }
    }
    if (tiles == 0 || __builtin_amdgcn_readfirstlane((int)s_bad) == 0) return;

    // ---- some V is no number, and not all rows see it: the wave's rows one by one,
    // 64 keys at a time (a lane its key's score, then two channels of every key's
    // value that the row sees) ----
    __builtin_amdgcn_s_waitcnt(0);   // the stores above come first
    constexpr int kCh = D / 64;      // channels of a lane
    for (int rr = 0; rr < 32 && r_wave + rr < n_rows; ++rr) {
        const int r1 = r_wave + rr, qi1 = (int)p.gqa.div((uint32_t)r1);
        const int head1 = kvh * G + (r1 - qi1 * G);
        const long q_row1 = (PREFIX ? (long)qi1 : (long)ft.row0 + qi1) * p.n_heads + head1;
        const int pos1 = PREFIX ? max(p.c.lens[qi1], 0) - 1 : ft.pos0 + qi1;
        const int old = oldest(pos1), lim = min(pos1 + 1, end);
        const float slope1 = p.s.slopes ? p.s.slopes[head1] * kLog2eF : 0.0f;
        float m = kNoMax, l = 0.0f, acc[kCh];
#pragma unroll
        for (int e = 0; e < kCh; ++e) acc[e] = 0.0f;
        for (int k0 = begin; k0 < lim; k0 += 64) {
            const int t = k0 + lane;
            long at = octet_offset<D>(p.c, table_row, kvh, t & ~7, end);
            const bool ok = t >= old && t < lim && at >= 0;
            at = ok ? at + (t & 7) * D : 0L;
            float dot = 0.0f;
            for (int d8 = 0; d8 < D; d8 += 8) {
                const u32x4 a = load16(p.q + q_row1 * D + d8), b = load16(p.c.k + at + d8);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = a[e], y = b[e];
                    dot = fmaf(Hf::to_f32((uint16_t)x), Hf::to_f32((uint16_t)y), dot);
                    dot = fmaf(Hf::to_f32((uint16_t)(x >> 16)), Hf::to_f32((uint16_t)(y >> 16)), dot);
                }
            }
            float s1 = EXACT ? capped_tanh(dot, p.s) * p.s.cap_log2
                             : p.s.cap_in != 0.0f ? capped(dot, p.s.cap_in, p.s.cap_log2) : dot * p.s.scale_log2;
            if (p.s.slopes) s1 = fmaf(-slope1, (float)(pos1 - t), s1);
            s1 = ok ? s1 : -INFINITY;
            float top = s1;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
            top = fmaxf(top, m);
            const float a = join_weight(m - top), p1 = __builtin_amdgcn_exp2f(s1 - top + kPShift);
            const float pt = ok ? (p1 < kMinWeight ? kMinWeight : p1) : 0.0f;   // (NaN stays)
            float sum = pt;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
            m = top;
            l = l * a + sum;
#pragma unroll
            for (int e = 0; e < kCh; ++e) acc[e] *= a;
            for (int j = 0; j < 64; ++j) {
                const float pj = __shfl(pt, j);
                const long vj = ((long)__shfl((int)(at >> 32), j) << 32) | (uint32_t)__shfl((int)(uint32_t)at, j);
                if (pj != 0.0f) {   // wave-uniform
#pragma unroll
                    for (int e = 0; e < kCh; ++e)
                        acc[e] = fmaf(pj, Hf::to_f32(p.c.v[vj + kCh * lane + e]), acc[e]);
                }
            }
        }
        if (as_part) {
            const long at = part_at(32 * wave + rr);
#pragma unroll
            for (int e = 0; e < kCh; ++e) p.part_o[at * D + kCh * lane + e] = acc[e];
            if (lane == 0) {
                p.part_ml[2 * at] = m;
                p.part_ml[2 * at + 1] = l;
            }
        } else {
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
            for (int e = 0; e < kCh; ++e)
                p.out[q_row1 * D + kCh * lane + e] = (uint16_t)Hf::pack(acc[e] * inv, 0.0f);
        }
    }
}

inline PagedFlashParams flash_params(const PagedLaunch& a) {
    PagedFlashParams p{};
    p.q = static_cast<const uint16_t*>(a.q);
    p.out = static_cast<uint16_t*>(a.out);
    p.c = paged_view(a);
    p.s = score_opts(a);
    p.cu = a.cu;
    p.rows = a.rows;
    p.per_round = (uint32_t)device_cu_count();
    p.n_heads = a.n_heads;
    p.gqa = FastDiv::of((uint32_t)(a.n_heads / a.n_kv_heads));
    return p;
}

}  // namespace llmik
