// The attention weight that a prompt's rows give each token:
//   weights[row(b), kvh, t] += sum over the sequence's last `observe` new rows i and
//                              the KV head's G query heads of softmax_t(s(i, t)).
// A softmax's weights are known once its row's maximum and sum are, so the scores are
// computed twice, by two kernels that keep one operand in registers and stream the
// other through LDS:
//   statistics: 128 rows (32 per wave) over the keys in tiles of 64. S^T = K Q^T gives
//     a lane one row's scores, so its maximum and sum stay in the lane. Where there are few
//     row tiles, their keys are cut into parts (Cutter).
//   sums: 128 keys (32 per wave) over the rows in tiles of 64. S^T = K Q^T again: a lane
//     has one row's m and 1 / l in registers and sums 2^(s - m) / l of its 16 keys; the
//     lanes are added once, behind the last tile. (S = Q K^T leaves a key's sum in one lane,
//     but reads 16 rows' m and 1 / l from LDS for 16 scores.)
// The parts of a cut row or key tile are joined, in order, by the last of its workgroups to
// arrive: nothing depends on timing. Where a sequence's recorded rows are one row tile (the
// last 32 tokens of four heads, say), its pass over the keys is the sums' too: whole columns,
// no joins, the statistics' parts joined by those who need them.
//
// Measured (32 heads over 8 KV heads of 128, bf16): all rows of 4000 tokens 185 .. 193 us, with a cap
// 255 .. 265, of 8192 tokens 635 .. 655; the products alone, twice, are 104 us at a large matrix
// product's rate. The statistics' vector units work 86 % of the cycles (9.5 instructions a score
// with a cap, three of them transcendental at half rate), the sums' 70 %. The last 32 rows of
// four prompts of 4000 .. 8192 tokens 31 .. 36 us, K's 48 MB read twice: 3 TB/s with two launches,
// their look-ups and the hand-off of the statistics. Three prompts of 17 .. 150 tokens 14: the two
// chains of launch, lengths, pages, keys.
#include "paged_flash.hpp"

namespace llmik {

constexpr int kPwThreads = 256;
constexpr int kPwKeys = 128;     // of a workgroup of the sums
constexpr int kPwTile = 64;      // rows or keys of a streamed tile

struct PromptWeightsParams {
    PagedFlashParams f;          // target, least and slots: the statistics' cuts
    f32x2* stats;                // [n_kv_heads, rows, G]: (maximum, 1 / sum); where that is no number, (that, 1)
    uint32_t* counters;          // of the cut tiles [slots / 2, n_kv_heads], zero between calls
    uint32_t* sum_counters;      // [sum_items, n_kv_heads]
    WeightsView w;
    float* part_sum;             // [2 sum_items, n_kv_heads, kPwKeys]
    int sum_items;               // workgroups of the sums for a KV head
    double sum_rate;             // 1 / sum_items
};

namespace {

// How scores become exponents (see paged_flash): sc * mult + add, after `score`.
template <bool EXACT>
struct ScoreForm {
    bool cap, modified;
    float mult, add;
    __device__ __forceinline__ explicit ScoreForm(const ScoreOpts& s) {
        cap = s.cap_in != 0.0f;
        modified = s.slopes != nullptr || (!cap && s.scale_log2 <= 0.0f);
        mult = modified ? 1.0f : EXACT ? s.cap_log2 : cap ? 2.0f * s.cap_log2 : s.scale_log2;
        add = cap && !modified && !EXACT ? s.cap_log2 : 0.0f;
    }
    // N scores as they come from the products; bias(e): the slope times the distance of score e.
    template <int N, typename B>
    __device__ __forceinline__ void apply(const ScoreOpts& s, float (&sc)[N], B bias) const {
        if constexpr (EXACT) {
#pragma unroll
            for (int e = 0; e < N; ++e) sc[e] = capped_tanh(sc[e], s);
        } else if (cap) {
#pragma unroll
            for (int e = 0; e < N; ++e) sc[e] = capped_part(sc[e], s.cap_in);
        }
        if (modified) {
            const float by = EXACT ? s.cap_log2 : cap ? 2.0f * s.cap_log2 : s.scale_log2;
            const float plus = cap && !EXACT ? s.cap_log2 : 0.0f;
#pragma unroll
            for (int e = 0; e < N; ++e) sc[e] = fmaf(sc[e], by, plus);
            if (s.slopes) {
#pragma unroll
                for (int e = 0; e < N; ++e) sc[e] -= bias(e);
            }
        }
    }
};

// 16-byte chunk slots of a tile's row in LDS are permuted by the row's number.
template <int D>
__device__ __forceinline__ int swizzle(int row) { return D == 128 ? row & 15 : row & 7; }

}  // namespace

// What a pass of 128 rows over their keys is for: their statistics, with the parts joined or
// (where the sums join them) left, or the sums.
enum class Pass { kStats, kStatParts, kSums };

// What a workgroup keeps in LDS beside three tiles of K; the sums' only but for `last`.
struct PassLds {
    float by[kPfRows], inv[kPfRows], slope[kPfRows];   // of the rows
    int pos[kPfRows];
    float sum[2][4][kPwTile];                          // a tile's keys', of each wave
    uint32_t last;
};

template <bool BF, int D, bool EXACT, Pass PASS>
__device__ __forceinline__ void row_pass(const PromptWeightsParams& pw, uint8_t* s_k0, uint8_t* s_k1, uint8_t* s_k2,
                                         PassLds& s) {
    using Hf = Half16<BF>;
    constexpr int KS = D / 16, CPR = D / 8, kRowBytes = 2 * D;
    constexpr int kCopies = 16 * CPR / 64, kRowsPerCopy = 64 / CPR;
    const PagedFlashParams& p = pw.f;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, h = lane >> 5, n = lane & 31;
    const int kvh = (int)(blockIdx.x % (uint32_t)p.c.n_kv_heads), G = (int)p.gqa.d;
    // Of the workgroups that run at once, one per CU and turn, every other turn's order is reversed: a CU's
    // then have about the same work together as another's.
    uint32_t item = blockIdx.x / (uint32_t)p.c.n_kv_heads;
    const uint32_t turn_items = max(p.per_round / (uint32_t)p.c.n_kv_heads, 1u), turn_no = item / turn_items;
    if (turn_no & 1u && (turn_no + 1) * turn_items <= gridDim.x / (uint32_t)p.c.n_kv_heads)
        item = (2 * turn_no + 1) * turn_items - 1 - item;
    CutItem ft{};
    auto sequence = [&](int b, CutItem& s) { cut_sequence(p, b, s); };
    const Cutter<decltype(sequence)> cutter(p, p.target, p.least, sequence);
    if (!cutter.find(item, ft)) return;
    if (ft.parts > 1 && (part_slot(ft, ft.parts - 1) >= p.slots || ft.cut >= p.slots / 2)) return;   // (the workspace's end)

    const int n_rows = ft.rows * G;
    const int r0 = ft.tile * kPfRows, r_wave = r0 + 32 * wave;
    const bool live = r_wave < n_rows;
    const int r = min(r_wave + n, n_rows - 1);
    const int qi = (int)p.gqa.div((uint32_t)r);
    const int head = kvh * G + (r - qi * G);
    const long q_row = ((long)ft.row0 + qi) * p.n_heads + head;
    const long st_row = ((long)kvh * p.rows + ft.row0) * G;   // of the sequence's first row
    const int pos = ft.ctx + qi;
    auto pos_of = [&](int row) { return ft.ctx + (int)p.gqa.div((uint32_t)min(row, n_rows - 1)); };
    const int pos_lo = __builtin_amdgcn_readfirstlane(pos_of(r_wave));
    const int pos_hi = __builtin_amdgcn_readfirstlane(pos_of(r_wave + 31));
    const int wg_lo = __builtin_amdgcn_readfirstlane(pos_of(r0));
    const int wg_hi = __builtin_amdgcn_readfirstlane(pos_of(r0 + kPfRows - 1));
    auto oldest = [&](int at) { return oldest_key(p.s, at); };
    // The part's keys that some row sees.
    const int part0 = ft.begin + ft.part * ft.part_tiles * kPwTile;
    const int begin = max(part0, oldest(wg_lo) / kPwTile * kPwTile);
    const int end = min(min(ft.end, wg_hi + 1), part0 + ft.part_tiles * kPwTile);
    const int tiles = end > begin ? (end - begin + kPwTile - 1) / kPwTile : 0;
    const int full_lo = (oldest(pos_hi) - begin + kPwTile - 1) >> 6;
    const int full_hi = (min(end, pos_lo + 1) - begin) >> 6;
    const int seen_lo = (oldest(pos_lo) - begin) >> 6;
    const int seen_hi = live ? ((pos_hi - begin) >> 6) + 1 : INT_MIN;
    [[maybe_unused]] float* const weights = PASS == Pass::kSums ? weights_of(pw.w, ft.b, kvh) : nullptr;
    if (PASS == Pass::kSums && (weights == nullptr || tiles == 0)) return;

    // ---- copies, as paged_flash's: wave w brings tokens 16 w .. + 15 of every tile ----
    const int* const table_row = p.c.table + (long)ft.b * p.c.max_pages;
    auto token_of = [&](int i0) { return begin + kPwTile * (i0 + (lane >> 3)) + 8 * (lane & 7); };
    auto look_up = [&](int i0) { return octet_offset<D>(p.c, table_row, kvh, token_of(i0), end); };
    int at_lo = 0, at_hi = 0, at_bytes = 0;
    uint64_t batch_gone = 0;
    auto adopt = [&](long off, int i0) {
        const bool gone = off < 0;
        const long at = gone ? 0L : 2 * off;
        at_lo = (int)(uint32_t)at;
        at_hi = (int)(at >> 32);
        at_bytes = gone ? 0 : min(max(end - token_of(i0), 0), 8) * kRowBytes;
        batch_gone = __ballot(gone);
    };
    long off_next = -1;
    u32x4 qb[KS];
    if (tiles > 0) adopt(look_up(0), 0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qb[ks] = load16(p.q + q_row * D + 16 * ks + 8 * h);
    const float slope = p.s.slopes ? p.s.slopes[head] * kLog2eF : 0.0f;
    if (tiles > 8) off_next = look_up(8);
    const int crow = lane / CPR, cslot = lane % CPR;
    uint32_t gone_next = 0, gone_now = 0;   // of the last tile requested, of the one before
    auto copy_tile = [&](uint8_t* dst, int i) {   // (where there is no tile i nothing is read, but counted)
        if ((i & 7) == 0 && i) {
            adopt(off_next, i);
            off_next = i + 8 < tiles ? look_up(i + 8) : -1L;
        }
        const int l0 = 8 * (i & 7);
        gone_next = (uint32_t)(batch_gone >> l0) & 255u;
        auto octet = [&](int l) {
            const long at = ((long)__builtin_amdgcn_readlane(at_hi, l) << 32) |
                            (uint32_t)__builtin_amdgcn_readlane(at_lo, l);
            return make_buffer_rsrc(reinterpret_cast<const uint8_t*>(p.c.k) + at,
                                    (uint32_t)__builtin_amdgcn_readlane(at_bytes, l));
        };
        const __amdgpu_buffer_rsrc_t rk0 = octet(l0 + 2 * wave), rk1 = octet(l0 + 2 * wave + 1);
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
            const int row = kRowsPerCopy * c + crow, trow = 16 * wave + row;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                (kRowsPerCopy * c) / 8 ? rk1 : rk0,
                (__attribute__((address_space(3))) void*)(dst + (16 * wave + kRowsPerCopy * c) * kRowBytes), 16,
                (row & 7) * kRowBytes + 16 * (cslot ^ swizzle<D>(trow)), 0, 0, 0);
        }
    };

    const ScoreForm<EXACT> form(p.s);
    float m_run = kNoMax, l_run = 0.0f;   // of row n, this lane's tokens
    if (tiles > 0) {   // (requested before the rows' statistics are)
        copy_tile(s_k0, 0);
        gone_now = gone_next;
        copy_tile(s_k1, 1);
    }
    [[maybe_unused]] float by_row[16], inv_row[16];   // the sums: of rows 8 (e / 4) + 4 h + e % 4 of the wave
    if constexpr (PASS == Pass::kSums) {
        // Two threads a row join its parts (every other one each, eight requested at a time).
        const int row = tid >> 1, rj = r0 + row, rc = min(rj, n_rows - 1), qj = (int)p.gqa.div((uint32_t)rc);
        float m = kNoMax, inv = 0.0f;
        if (ft.parts == 1) {
            const f32x2 st = pw.stats[st_row + rc];
            m = st[0];
            inv = st[1];
        } else {
            float l = 0.0f;
            constexpr int kBatch = 8;
            for (int u0 = tid & 1; u0 < ft.parts; u0 += 2 * kBatch) {
                f32x2 ml[kBatch];
#pragma unroll
                for (int u = 0; u < kBatch; ++u)
                    ml[u] = *reinterpret_cast<const f32x2*>(
                        p.part_ml + 2 * part_row(p, part_slot(ft, min(u0 + 2 * u, ft.parts - 1)), kvh, row));
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    if (u0 + 2 * u < ft.parts) {
                        const float top = fmaxf(m, ml[u][0]);
                        l = l * __builtin_amdgcn_exp2f(m - top) + ml[u][1] * __builtin_amdgcn_exp2f(ml[u][0] - top);
                        m = top;
                    }
                }
            }
            const float m2 = dpp_f32<kDppQuadXor1>(m), l2 = dpp_f32<kDppQuadXor1>(l), top = fmaxf(m, m2);
            l = l * __builtin_amdgcn_exp2f(m - top) + l2 * __builtin_amdgcn_exp2f(m2 - top);
            m = top;
            inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        }
        if ((tid & 1) == 0) {
            s.by[row] = form.add - m;
            s.inv[row] = rj < n_rows ? inv : 0.0f;
            s.pos[row] = rj < n_rows ? ft.ctx + qj : INT_MIN;   // (sees no key)
            if (p.s.slopes) s.slope[row] = p.s.slopes[kvh * G + (rc - qj * G)] * kLog2eF;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            by_row[e] = s.by[32 * wave + 8 * (e >> 2) + 4 * h + (e & 3)];
            inv_row[e] = s.inv[32 * wave + 8 * (e >> 2) + 4 * h + (e & 3)];
        }
    }
    const uint32_t k_row = (uint32_t)(n * kRowBytes);
    const uint32_t k_sw = (uint32_t)((h ^ swizzle<D>(n)) * 16);
    auto statistics = [&](const uint8_t* sk, int i, uint32_t gone) {
        const int t0 = begin + kPwTile * i, tk = t0 + 4 * h;
        float sc[32];
        u32x4 ka[2][KS];   // the keys' operands, eight products ahead
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
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[16 * blk + e] = acc[e];
        }
        form.apply(p.s, sc, [&](int e) { return slope * (float)(pos - (tk + 8 * (e >> 2) + (e & 3))); });
        if (gone || i < full_lo || i >= full_hi) {   // wave-uniform
            const int old = oldest(pos), lim = min(pos + 1, end);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const int tok = tk + 8 * (e >> 2) + (e & 3);
                if (tok < old || tok >= lim || ((gone >> (e >> 2)) & 1u)) sc[e] = -INFINITY;
            }
        }
        float top = sc[0];
#pragma unroll
        for (int e = 1; e < 32; ++e) top = fmaxf(top, sc[e]);
        const float m_new = fmaxf(m_run, fmaf(top, form.mult, form.add));
        l_run *= __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        const float by = form.add - m_new;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 32; ++e) sum[e & 3] += __builtin_amdgcn_exp2f(fmaf(sc[e], form.mult, by));
        l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    };
    // The sums: S = Q K^T, a lane has key n of each block and 16 of the wave's rows.
    auto sums = [&](const uint8_t* sk, int i, uint32_t gone) {
        const int t0 = begin + kPwTile * i;
        const bool masked = gone || i < full_lo || i >= full_hi || r_wave + 32 > n_rows;   // wave-uniform
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            f32x16 acc;
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                acc = Hf::mfma32(qb[ks],
                                 *reinterpret_cast<const u32x4*>(sk + k_row + 32 * blk * kRowBytes + (k_sw ^ (32u * ks))),
                                 acc);
            float sc[16], sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const int key = t0 + 32 * blk + n;
            auto row_of = [&](int e) { return 32 * wave + 8 * (e >> 2) + 4 * h + (e & 3); };
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[e] = acc[e];
            form.apply(p.s, sc, [&](int e) { return s.slope[row_of(e)] * (float)(s.pos[row_of(e)] - key); });
            if (!masked) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    sum[e & 3] = fmaf(__builtin_amdgcn_exp2f(fmaf(sc[e], form.mult, by_row[e])), inv_row[e], sum[e & 3]);
            } else {
                const bool key_ok = key < end && !((gone >> (4 * blk + (n >> 3))) & 1u);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int at = s.pos[row_of(e)];
                    const float x = __builtin_amdgcn_exp2f(fmaf(sc[e], form.mult, by_row[e]));
                    if (key_ok && at >= key && at - key < p.s.window) sum[e & 3] = fmaf(x, inv_row[e], sum[e & 3]);
                }
            }
            const float all = xor32_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
            if (h == 0) s.sum[i & 1][wave][32 * blk + n] = all;
        }
    };
    // The waves' sums of tile i, added to the weights by the first wave.
    float weight = 0.0f;   // of the tile before the one computed
    auto record = [&](int i) {
        const int key = begin + kPwTile * i + lane;
        const float all = (s.sum[i & 1][0][lane] + s.sum[i & 1][1][lane]) + (s.sum[i & 1][2][lane] + s.sum[i & 1][3][lane]);
        if (key < min(end, pw.w.max_len)) weights[key] = weight + all;
    };
    // Two tiles ahead: a tile's copies are complete once at most the next one's are outstanding (loads
    // complete in order), and for the whole workgroup behind the barrier, where the buffer of the tile
    // before is free.
    auto turn = [&](uint8_t* cur, uint8_t* free, int i) {
        if constexpr (kCopies == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
        if constexpr (PASS == Pass::kSums) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");
        const uint32_t gone = gone_now;
        gone_now = gone_next;
        if constexpr (PASS == Pass::kSums) {
            if (wave == 0) {   // (before the copies, which the next wait counts)
                if (i > 0) record(i - 1);
                weight = weights[min(begin + kPwTile * i + lane, min(end, pw.w.max_len) - 1)];
            }
        }
        copy_tile(free, i + 2);
        const bool sees = i >= seen_lo && i < seen_hi;
        if constexpr (PASS != Pass::kSums) {
            if (sees) statistics(cur, i, gone);
        } else {
            if (sees) sums(cur, i, gone);
            else s.sum[i & 1][wave][lane] = 0.0f;
        }
    };
    static_assert(kCopies == 4 || kCopies == 2, "the wait counts a tile's copies");
    for (int i = 0; i < tiles; i += 3) {
        turn(s_k0, s_k2, i);
        if (i + 1 < tiles) turn(s_k1, s_k0, i + 1);
        if (i + 2 < tiles) turn(s_k2, s_k1, i + 2);
    }
    __builtin_amdgcn_s_waitcnt(0);   // no copy into LDS outlives the workgroup
    if constexpr (PASS == Pass::kSums) {
        __syncthreads();
        if (wave == 0) record(tiles - 1);
        return;
    }

    const float m_row = xor32_max(m_run);
    const float l_row = xor32_sum(l_run * __builtin_amdgcn_exp2f(m_run - m_row));
    auto store = [&](long at, float m, float l) {
        pw.stats[at] = l != l ? f32x2{l, 1.0f} : f32x2{m, l > 0.0f ? 1.0f / l : 0.0f};
    };
    const bool mine = h == 0 && r_wave + n < n_rows;
    if (ft.parts == 1) {
        if (mine) store(st_row + r, m_row, l_row);
        return;
    }
    float* const to = p.part_ml + 2 * part_row(p, part_slot(ft, ft.part), kvh, 32 * wave + n);
    if constexpr (PASS == Pass::kStatParts) {
        if (mine) *reinterpret_cast<f32x2*>(to) = f32x2{m_row, l_row};
        return;
    }
    if (mine) {
        const uint64_t ml = (uint64_t)__float_as_uint(l_row) << 32 | __float_as_uint(m_row);
        __hip_atomic_store(reinterpret_cast<uint64_t*>(to), ml, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    publish_wait();
    __syncthreads();
    uint32_t* const counter = pw.counters + (long)ft.cut * p.c.n_kv_heads + kvh;
    if (tid == 0) s.last = arrive_last(counter, (uint32_t)ft.parts) ? 1u : 0u;
    __syncthreads();
    if (s.last == 0) return;
    if (tid == 0) *counter = 0u;   // for the next call
    const int rj = r0 + tid;
    if (tid >= kPfRows || rj >= n_rows) return;
    float m = kNoMax, l = 0.0f;
    constexpr int kBatch = 8;   // requested at a time
    for (int u0 = 0; u0 < ft.parts; u0 += kBatch) {
        uint64_t ml[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const uint32_t slot = part_slot(ft, min(u0 + u, ft.parts - 1));
            ml[u] = __hip_atomic_load(reinterpret_cast<uint64_t*>(p.part_ml + 2 * part_row(p, slot, kvh, tid)),
                                      __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const float mu = __uint_as_float((uint32_t)ml[u]), lu = __uint_as_float((uint32_t)(ml[u] >> 32));
            const float top = fmaxf(m, mu);
            if (u0 + u < ft.parts) l = l * __builtin_amdgcn_exp2f(m - top) + lu * __builtin_amdgcn_exp2f(mu - top);
            m = top;   // (a part that is repeated has no greater maximum)
        }
    }
    store(st_row + rj, m, l);
}

template <bool BF, int D, bool EXACT, Pass PASS>
__global__ __launch_bounds__(kPwThreads, 3) void paged_row_pass_kernel(PromptWeightsParams pw) {
    __shared__ __attribute__((aligned(16))) uint8_t s_k0[kPwTile * 2 * D], s_k1[kPwTile * 2 * D];
    __shared__ __attribute__((aligned(16))) uint8_t s_k2[kPwTile * 2 * D];
    __shared__ __attribute__((aligned(16))) PassLds s;
    row_pass<BF, D, EXACT, PASS>(pw, s_k0, s_k1, s_k2, s);
}

// The work of the sums is a list of (key tile of kPwKeys, row tile of kPwTile) pairs, key tile by
// key tile, of which every workgroup of a KV head takes the same number, one after the other: where
// that ends inside a key tile the next workgroup goes on. Key tile i of a sequence is seen by row
// tiles first(i) .. last(i) - 1, which move by 2 G from one to the next until they reach the rows'
// end, so that a sequence's pairs up to any key tile are a closed sum. (Equal cuts of all row tiles,
// of which a causal prompt's key tiles see half: us, 4000 tokens 208 against 189, two of 1500
// 91, 77. Short ones with 1, 2, 4 pairs for a workgroup at least: 100 tokens 18.4, 19.6, 22.2, 200
// 19.4, 23.7, 26.5, 600 27.1, 27.1, 30.9, 8 of 150 25.1, 24.3, 26.9.)
struct KeySeq {
    int b, row0, rows, ctx;   // as CutItem's
    int begin, end;           // the keys that are recorded
    int keys, row_tiles;      // key tiles, row tiles
    long lo, hi;              // first(0) and last(0), which may lie outside the rows
    int at_lo, at_hi;         // key tiles from which on lo + 2 G i >= 0, hi + 2 G i >= row_tiles (or `keys`)

    __device__ __forceinline__ int first(int i, int G) const { return (int)max(lo + 2L * G * i, 0L); }
    __device__ __forceinline__ int last(int i, int G) const { return (int)min(hi + 2L * G * i, (long)row_tiles); }
    // The pairs of the first n key tiles.
    __device__ __forceinline__ long pairs(int n, int G) const {
        const long below = max(n - at_lo, 0), moving = min(n, at_hi);
        return moving * (hi + G * (moving - 1)) + (n - moving) * row_tiles - below * (lo + G * (at_lo + n - 1L));
    }
};

__device__ __forceinline__ void key_sequence(const PromptWeightsParams& pw, int b, KeySeq& s) {
    const PagedFlashParams& p = pw.f;
    const int G = (int)p.gqa.d;
    CutItem t;
    cut_sequence(p, b, t);
    s.b = b;
    s.row0 = t.row0;
    s.rows = t.rows;
    s.ctx = t.ctx;
    s.begin = t.begin;
    s.end = min(min(t.end, pw.w.max_len), t.ctx + t.rows);
    s.row_tiles = (int)((uint32_t)(t.rows * G + kPwTile - 1) / kPwTile);
    // The first key lies d tokens behind the first row, and `reach` in front of the first that sees none of its tile.
    const long d = (long)s.begin - s.ctx, reach = d + kPwKeys - 1 + p.s.window;
    s.lo = (d * G) >> 6;
    s.hi = min((reach * G + kPwTile - 1) >> 6, (long)s.row_tiles);
    const bool recorded = t.rows > 0 && s.end > s.begin && s.hi > 0 && weights_of(pw.w, b, 0) != nullptr;
    s.keys = recorded ? (s.end - s.begin + kPwKeys - 1) / kPwKeys : 0;
    auto tiles_to = [&](long keys) { return (int)min(max(keys + kPwKeys - 1, 0L) / kPwKeys, (long)s.keys); };
    s.at_lo = tiles_to(-d);
    s.at_hi = tiles_to(t.rows - reach);
}

template <bool BF, int D, bool EXACT>
__global__ __launch_bounds__(kPwThreads, 3) void paged_key_sums_kernel(PromptWeightsParams pw) {
    using Hf = Half16<BF>;
    constexpr int KS = D / 16, CPR = D / 8, kRowBytes = 2 * D;
    constexpr int kCopies = 16 * CPR / 64, kRowsPerCopy = 64 / CPR;
    __shared__ __attribute__((aligned(16))) uint8_t s_q0[kPwTile * kRowBytes], s_q1[kPwTile * kRowBytes];
    __shared__ uint32_t s_last;
    __shared__ KeySeq s_seq[64];   // the last of sequences per * l .. per * l + per - 1
    __shared__ long s_upto[64];    // the pairs up to its end
    __shared__ __attribute__((aligned(16))) float s_by[2][kPwTile], s_inv[2][kPwTile], s_slope[2][kPwTile];
    __shared__ __attribute__((aligned(16))) int s_pos[2][kPwTile];
    const PagedFlashParams& p = pw.f;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, h = lane >> 5, n = lane & 31;
    const int G = (int)p.gqa.d;
    const ScoreForm<EXACT> form(p.s);
    const uint32_t q_at = (uint32_t)(n * kRowBytes);
    const uint32_t q_sw = (uint32_t)((h ^ swizzle<D>(n)) * 16);
    const int kvh = (int)(blockIdx.x % (uint32_t)p.c.n_kv_heads), item = (int)(blockIdx.x / (uint32_t)p.c.n_kv_heads);
    const int per = (p.c.batch + 63) / 64;
    if (wave == 0) {
        long upto = 0;
        KeySeq s{};
        for (int b = min(lane * per, p.c.batch); b < min(lane * per + per, p.c.batch); ++b) {
            key_sequence(pw, b, s);
            upto += s.pairs(s.keys, G);
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const long other = __shfl_up(upto, d);
            if (lane >= d) upto += other;
        }
        s_seq[lane] = s;
        s_upto[lane] = upto;
    }
    __syncthreads();
    auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    auto uniform64 = [&](long x) { return (long)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x); };
    const long pairs = uniform64(s_upto[63]);
    long chunk = (long)((double)pairs * pw.sum_rate);
    if (chunk * pw.sum_items < pairs) ++chunk;
    chunk = uniform64(chunk);
    const long stop = min(pairs, (item + 1) * chunk);
    for (long at = item * chunk; at < stop;) {
        // ---- the pair `at`: its sequence, its key tile, its row tile ----
        const int lane_at = __popcll(__ballot(s_upto[lane] <= at));
        KeySeq t = s_seq[lane_at];
        long into = at;   // the pair's number among its sequence's
        if (per == 1) into -= s_upto[lane_at] - t.pairs(t.keys, G);
        else {
            into -= lane_at > 0 ? s_upto[lane_at - 1] : 0L;
            for (int b = lane_at * per;; ++b) {   // ends: the lane's sequences hold the pair
                key_sequence(pw, b, t);
                const long n = t.pairs(t.keys, G);
                if (into < n || b + 1 >= min(lane_at * per + per, p.c.batch)) break;
                into -= n;
            }
        }
        into = uniform64(into);
        t.b = uniform(t.b);
        t.row0 = uniform(t.row0);
        t.rows = uniform(t.rows);
        t.ctx = uniform(t.ctx);
        t.begin = uniform(t.begin);
        t.end = uniform(t.end);
        t.keys = uniform(t.keys);
        t.row_tiles = uniform(t.row_tiles);
        t.lo = uniform64(t.lo);
        t.hi = uniform64(t.hi);
        t.at_lo = uniform(t.at_lo);
        t.at_hi = uniform(t.at_hi);
        int tile = 0;
        for (int n = t.keys; n > 1;) {   // the last with pairs(tile) <= into, among n: 64 of them at once
            const int step = (n + 63) / 64, probe = min((lane + 1) * step, n);
            const int more = __popcll(__ballot(probe < n && t.pairs(tile + probe, G) <= into)) * step;
            tile += more;
            n = min(n - more, step);
        }
        const int rt0 = t.first(tile, G), of_tile = t.last(tile, G) - rt0;
        const int before = (int)(into - t.pairs(tile, G));
        const int tiles = (int)min((long)(of_tile - before), stop - at), after = of_tile - before - tiles;
        at += tiles;
        // Its parts: this one, and those of the workgroups before and behind (all but the last take `chunk`).
        const uint32_t length = (uint32_t)min(chunk, 1L << 30);
        const int part = (int)quick_ceil((uint32_t)before, length);
        const int parts = part + 1 + (int)quick_ceil((uint32_t)after, length);
        const int item0 = item - part;   // that of the first
        const int n_rows = t.rows * G;
        const int key0 = t.begin + kPwKeys * tile, key_end = min(t.end, key0 + kPwKeys);
        const int r_lo = kPwTile * (rt0 + before);
        const int r_hi = min((int)min((long)t.rows, (long)key_end - 1 + p.s.window - t.ctx) * G, r_lo + kPwTile * tiles);

        // ---- the wave's keys ----
        const int key_w = key0 + 32 * wave, key = key_w + n;
        const int* const table_row = p.c.table + (long)t.b * p.c.max_pages;
        const long off = octet_offset<D>(p.c, table_row, kvh, key & ~7, key_end);
        const bool key_ok = off >= 0 && key < key_end;
        u32x4 kb[KS];
        {
            const uint16_t* from = p.c.k + (off < 0 ? 0L : off + (key & 7) * D) + 8 * h;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) kb[ks] = load16(from + 16 * ks);
        }

        // Lane (h, n < 16) adds key `own` of the wave's in the end. Its weight so far (read by all of a key tile's
        // parts: the last one adds).
        const int own = 8 * ((n & 15) >> 2) + 4 * h + (n & 3);
        const uint32_t keys_ok = (uint32_t)__ballot(key_ok);
        float* to = nullptr;
        float weight = 0.0f;
        if (n < 16 && keys_ok >> own & 1u && key_w + own < pw.w.max_len) {
            to = weights_of(pw.w, t.b, kvh);
            if (to != nullptr) weight = *(to += key_w + own);
        }

        // ---- rows of a tile: wave w brings 16 w .. + 15; threads 0 .. 63 their numbers ----
        const uint16_t* const q_seq = p.q + ((long)t.row0 * p.n_heads + kvh * G) * D;
        const f32x2* const st_seq = pw.stats + ((long)kvh * p.rows + t.row0) * G;
        const int crow = lane / CPR, cslot = lane % CPR;
        // The next tile's first row: its query token, its head. Where G divides a tile the rows lie alike in all
        // tiles (and the look-up of their places was a fifth of the vector work).
        const int step_q = (int)p.gqa.div((uint32_t)kPwTile), step_head = kPwTile - step_q * G;
        int next_q = __builtin_amdgcn_readfirstlane((int)p.gqa.div((uint32_t)r_lo)), next_head = r_lo - next_q * G;
        uint32_t place[kCopies];
        auto copy_tile = [&](uint8_t* dst, int i) {
            if (i >= tiles) return;
            if (i == 0 || step_head != 0) {
#pragma unroll
                for (int c = 0; c < kCopies; ++c) {
                    const int trow = 16 * wave + kRowsPerCopy * c + crow, r = next_head + trow;
                    const int qi = (int)p.gqa.div((uint32_t)r);
                    place[c] = (uint32_t)(qi * p.n_heads + (r - qi * G)) * kRowBytes + 16u * (uint32_t)(cslot ^ swizzle<D>(trow));
                }
            }
            // (Rows behind the sequence's last token lie outside the buffer's range: zeros.)
            const long left = (long)(t.rows - next_q) * p.n_heads * kRowBytes;
            const __amdgpu_buffer_rsrc_t rq = make_buffer_rsrc(q_seq + (long)next_q * p.n_heads * D,
                                                               (uint32_t)min(left, 0xFFFFFFFFl));
#pragma unroll
            for (int c = 0; c < kCopies; ++c)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rq, (__attribute__((address_space(3))) void*)(dst + (16 * wave + kRowsPerCopy * c) * kRowBytes), 16,
                    (int)place[c], 0, 0, 0);
            next_q += step_q;
            next_head += step_head;
            if (next_head >= G) {
                next_head -= G;
                ++next_q;
            }
        };
        f32x2 st = {0.0f, 0.0f};
        auto load_stats = [&](int i) {
            if (tid < kPwTile && i < tiles) st = st_seq[min(r_lo + kPwTile * i + tid, n_rows - 1)];
        };
        auto put_stats = [&](int i) {
            if (tid < kPwTile && i < tiles) {
                const int r = r_lo + kPwTile * i + tid, rc = min(r, n_rows - 1);
                const int qi = (int)p.gqa.div((uint32_t)rc), at = i & 1;
                s_by[at][tid] = form.add - st[0];
                s_inv[at][tid] = r < r_hi ? st[1] : 0.0f;
                s_pos[at][tid] = r < r_hi ? t.ctx + qi : INT_MIN;   // (sees no key)
                if (p.s.slopes) s_slope[at][tid] = p.s.slopes[kvh * G + (rc - qi * G)] * kLog2eF;
            }
        };

        float sum[16] = {};   // of keys 8 (e / 4) + 4 h + e % 4, rows n of the blocks
        auto compute = [&](const uint8_t* sq, int i) {
            const int r0 = r_lo + kPwTile * i, at = i & 1;
            const int pos_lo = t.ctx + (int)p.gqa.div((uint32_t)r0);
            const int pos_hi = t.ctx + (int)p.gqa.div((uint32_t)min(r0 + kPwTile, r_hi) - 1u);
            if (pos_hi < key_w || key_w >= key_end) return;   // wave-uniform
            const bool full = r0 + kPwTile <= r_hi && pos_lo >= key_w + 31 && pos_hi - key_w < p.s.window;
            // The rows' operands, eight products ahead.
            u32x4 qa[2][KS];
            auto load_q = [&](int blk, int ks) {
                qa[blk][ks] = *reinterpret_cast<const u32x4*>(sq + q_at + 32 * blk * kRowBytes + (q_sw ^ (32u * ks)));
            };
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) load_q(0, ks);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                f32x16 acc;
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    acc = Hf::mfma32(kb[ks], qa[blk][ks], acc);
                    if (blk == 0) load_q(1, ks);
                    __builtin_amdgcn_sched_barrier(0);
                }
                const int row = 32 * blk + n, key0 = key_w + 4 * h;
                const float by = s_by[at][row], inv = s_inv[at][row];
                float sc[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[e] = acc[e];
                form.apply(p.s, sc, [&](int e) {
                    return s_slope[at][row] * (float)(s_pos[at][row] - (key0 + 8 * (e >> 2) + (e & 3)));
                });
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], form.mult, by));
                if (!full) {
                    const int pos = s_pos[at][row];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int k = key0 + 8 * (e >> 2) + (e & 3);
                        if (pos < k || pos - k >= p.s.window) sc[e] = 0.0f;
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) sum[e] = fmaf(sc[e], inv, sum[e]);
            }
        };
        auto turn = [&](uint8_t* cur, uint8_t* far, int i) {
            __builtin_amdgcn_s_waitcnt(0);
            asm volatile("s_barrier" ::: "memory");
            put_stats(i + 1);
            load_stats(i + 2);
            copy_tile(far, i + 1);
            compute(cur, i);
        };
        load_stats(0);
        copy_tile(s_q0, 0);
        put_stats(0);
        load_stats(1);
        for (int i = 0; i < tiles; i += 2) {
            turn(s_q0, s_q1, i);
            if (i + 1 < tiles) turn(s_q1, s_q0, i + 1);
        }
        // The rows' 32 classes together: a lane passes on the half of its keys that the other's bit of n names.
#pragma unroll
        for (int w = 8; w > 0; w >>= 1)
#pragma unroll
            for (int e = 0; e < w; ++e) {
                const float keep = n & w ? sum[e + w] : sum[e], give = n & w ? sum[e] : sum[e + w];
                sum[e] = keep + __shfl_xor(give, w);
            }
        const float all = sum[0] + __shfl_xor(sum[0], 16);
        if (parts == 1) {
            if (to != nullptr) *to = weight + all;
        } else {
            // The last of the key tile's workgroups to arrive adds its parts, in order.
            // A workgroup's last key tile, which the next one continues, has its odd slot, its first the even one.
            auto part_at = [&](int part, int i) {
                const long slot = 2L * (item0 + part) + (part == 0 ? 1 : 0);
                return pw.part_sum + (slot * p.c.n_kv_heads + kvh) * kPwKeys + i;
            };
            if (n < 16) publish_store(part_at(part, 32 * wave + own), all);
            publish_wait();
            __syncthreads();
            uint32_t* const counter = pw.sum_counters + (long)item0 * p.c.n_kv_heads + kvh;
            if (tid == 0) s_last = arrive_last(counter, (uint32_t)parts) ? 1u : 0u;
            __syncthreads();
            if (s_last != 0) {
                if (tid == 0) *counter = 0u;   // for the next call
                float sum = 0.0f;
                constexpr int kBatch = 8;   // requested at a time
                for (int u0 = 0; u0 < parts; u0 += kBatch) {
                    float x[kBatch];
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) x[u] = publish_load(part_at(min(u0 + u, parts - 1), 32 * wave + own));
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) sum += u0 + u < parts ? x[u] : 0.0f;
                }
                if (to != nullptr) *to = weight + sum;
            }
        }
        __builtin_amdgcn_s_waitcnt(0);   // no copy into LDS outlives the workgroup, and
        __syncthreads();   // the tiles are read before the next ones are copied
    }
}

// ---------------------------------------------------------------- host

namespace {

// Key tiles are cut for two workgroups per CU, into single tiles where there are few. us, the last 32 rows of four
// prompts of 4000 .. 8192 tokens for 1, 2, 3 workgroups 43, 36, 38, the last 16 of 2000 tokens with 1, 2, 4 tiles or
// more 15.0, 16.0, 19.6, the last 16 of 16 x 4000 for 1, 2, 3 85, 65, 62.
constexpr int kStatsPerCu = 2, kStatsLeast = 1;
// Three workgroups of the sums run on a CU at once.
constexpr int kSumsPerCu = 3;

struct PromptWeightsPlan {
    long row_tiles;
    int target, sum_items;
    bool one_tile;        // a sequence's recorded rows of a KV head are one row tile: its pass sums up whole columns
    uint32_t slots;
    size_t off_ml, off_stats, off_sum, bytes;
};

PromptWeightsPlan plan_prompt_weights(int batch, int rows, int n_heads, int n_kv_heads, int observe, int cus) {
    PromptWeightsPlan pl{};
    const long seen = observe > 0 ? std::min((long)rows, (long)batch * observe) : rows;
    const long all = seen * (n_heads / n_kv_heads);
    pl.row_tiles = std::min((all + (long)batch * (kPfRows - 1)) / kPfRows, all / kPfRows + std::min((long)batch, seen));
    pl.target = std::max(kStatsPerCu * cus / n_kv_heads, 1);
    pl.slots = 2u * (uint32_t)pl.target;
    pl.sum_items = std::max(kSumsPerCu * cus / n_kv_heads, 1);
    const long most = (observe > 0 ? std::min(rows, observe) : rows) * (long)(n_heads / n_kv_heads);   // of a sequence
    pl.one_tile = most <= kPfRows;
    // A counter for each cut tile: where they do not suffice (thousands of KV heads), nothing is cut.
    if ((long)(pl.target + pl.sum_items) * n_kv_heads > kMaxCounters) {
        pl.slots = 0;
        pl.sum_items = 1;
    }
    pl.off_ml = kCounterBytes;
    pl.off_stats = pl.off_ml + align_up((size_t)pl.slots * n_kv_heads * kPfRows * 2 * sizeof(float), 256);
    pl.off_sum = pl.off_stats + align_up((size_t)rows * n_heads * 2 * sizeof(float), 256);
    pl.bytes = pl.off_sum + 2 * (size_t)pl.sum_items * n_kv_heads * kPwKeys * sizeof(float);
    return pl;
}

template <bool BF, int D, bool EXACT>
void launch_prompt(const PromptWeightsParams& pw, const PromptWeightsPlan& pl, hipStream_t stream) {
    const int hkv = pw.f.c.n_kv_heads;
    const unsigned grid = (unsigned)((pl.row_tiles + pl.target) * hkv);
    if (pl.one_tile) {
        paged_row_pass_kernel<BF, D, EXACT, Pass::kStatParts><<<grid, kPwThreads, 0, stream>>>(pw);
        paged_row_pass_kernel<BF, D, EXACT, Pass::kSums><<<grid, kPwThreads, 0, stream>>>(pw);
        return;
    }
    paged_row_pass_kernel<BF, D, EXACT, Pass::kStats><<<grid, kPwThreads, 0, stream>>>(pw);
    paged_key_sums_kernel<BF, D, EXACT><<<(unsigned)(pl.sum_items * hkv), kPwThreads, 0, stream>>>(pw);
}

}  // namespace

size_t paged_prefill_weights_workspace(int batch, int rows, int n_heads, int n_kv_heads, int observe) {
    return plan_prompt_weights(batch, rows, n_heads, n_kv_heads, observe, device_cu_count()).bytes;
}

int launch_paged_prefill_weights(const PagedLaunch& a, const PagedWeights& w, int observe, hipStream_t stream) {
    const PromptWeightsPlan pl =
        plan_prompt_weights(a.batch, a.rows, a.n_heads, a.n_kv_heads, observe, device_cu_count());
    if (a.workspace == nullptr || a.workspace_bytes < pl.bytes)
        return set_error(LLMIK_ERR_WORKSPACE, "workspace too small (llmik_paged_prefill_weights_workspace_size)");
    PromptWeightsParams pw{};
    pw.f = flash_params(a);
    pw.f.splits = 1;
    pw.f.observe = observe > 0 ? observe : INT_MAX;
    pw.f.target = pl.target;
    pw.f.least = pl.slots > 0 ? kStatsLeast : kUncut;
    pw.f.slots = pl.slots;
    char* ws = static_cast<char*>(a.workspace);
    pw.counters = reinterpret_cast<uint32_t*>(ws);
    pw.sum_counters = pw.counters + (long)(pl.slots / 2) * a.n_kv_heads;
    pw.f.part_ml = reinterpret_cast<float*>(ws + pl.off_ml);
    pw.stats = reinterpret_cast<f32x2*>(ws + pl.off_stats);
    pw.part_sum = reinterpret_cast<float*>(ws + pl.off_sum);
    pw.w = weights_view(w, a.n_kv_heads);
    pw.sum_items = pl.sum_items;
    pw.sum_rate = 1.0 / pl.sum_items;
    auto go = [&](auto bf, auto exact) {
        constexpr bool BF = decltype(bf)::value, EXACT = decltype(exact)::value;
        if (a.head_dim == 128) launch_prompt<BF, 128, EXACT>(pw, pl, stream);
        else launch_prompt<BF, 64, EXACT>(pw, pl, stream);
    };
    using std::false_type;
    using std::true_type;
    const bool exact = pw.f.s.cap_x != 0.0f;
    if (a.bf16) exact ? go(true_type{}, true_type{}) : go(true_type{}, false_type{});
    else exact ? go(false_type{}, true_type{}) : go(false_type{}, false_type{});
    return check_launch();
}

}  // namespace llmik
