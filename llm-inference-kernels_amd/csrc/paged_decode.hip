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
#include "paged_common.hpp"

namespace llmik {

namespace {

constexpr int kPdThreads = 256;
constexpr int kPdWaves = 4;
constexpr float kPShift = 8.0f;   // p is held as 2^8 p: fp16 keeps its full precision down to 2^-22

struct PagedDecodeParams {
    const uint16_t* q;
    uint16_t* out;
    PagedView c;
    ScoreOpts s;
    int n_heads, gqa, n_chunks, chunk_heads;   // query heads per KV head, their chunks, heads of a chunk (<= 16)
    int first;            // keys before this position are not this kernel's (the shared prefix)
    const float* pre_o;   // the prefix's partials [n_kv_heads, batch * gqa, pre_splits, D] and (m, l)
    const float* pre_ml;
    int pre_splits;
    float* part_o;        // [2 * workgroups, chunk_heads, D]
    float* part_ml;       // [2 * workgroups, chunk_heads, 2]
    uint32_t* counters;   // [workgroups], zero between calls
    int min_share;        // tiles per workgroup at least
};

struct Slab {
    int b, kvh, chunk;
    int len, begin, end;      // the sequence's length, its live keys [begin, end)
    int tile0, tiles;         // first 32-token tile, tiles of the slab
    uint32_t start;           // the slab's first tile among all slabs' tiles
};

// Keys [begin, end) of sequence b and their 32-token tiles. Every sequence has
// one tile at least, so that its rows are written.
__device__ __forceinline__ void keys_of(const PagedDecodeParams& p, int len, int& begin, int& end, int& tiles) {
    len = max(len, 0);
    end = min(len, p.c.capacity);
    begin = max(max(len - p.s.window, 0), p.first);
    tiles = max((end + 31) / 32 - begin / 32, 1);
}

// One 32-token tile's K and V of a (sequence, KV head) in the operand order.
template <int D>
struct PagedTile {
    static constexpr int KS = D / 32, VEC = D / 16;
    u32x4 k[2][KS];
    uint32_t v[8][VEC / 2];
};

}  // namespace

template <bool BF, int D, bool UNI>
__global__ __launch_bounds__(kPdThreads, 2) void paged_decode_kernel(PagedDecodeParams p) {
    using Hf = Half16<BF>;
    constexpr int KS = D / 32, VEC = D / 16, VW = VEC / 2;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, g = lane >> 4, c = lane & 15;

    __shared__ uint32_t s_pre[kPdThreads + 1];
    __shared__ Slab s_slab;
    __shared__ uint32_t s_last;
    __shared__ __attribute__((aligned(16))) float s_o[kPdWaves][16][D + 4];
    __shared__ float s_m[kPdWaves][16], s_l[kPdWaves][16];

    // ---- the shares: running totals of the sequences' tiles ----
    const int per_thread = (p.c.batch + kPdThreads - 1) / kPdThreads;
    const int slabs = p.c.n_kv_heads * p.n_chunks;   // of one sequence
    const int b0 = min(tid * per_thread, p.c.batch), b1 = min(b0 + per_thread, p.c.batch);
    uint32_t mine = 0;
    for (int b = b0; b < b1; ++b) {
        int begin, end, tiles;
        keys_of(p, p.c.lens[b], begin, end, tiles);
        mine += (uint32_t)(tiles * slabs);
    }
    const uint32_t total = block_totals(mine, s_pre);
    uint32_t share = max((total + gridDim.x - 1) / gridDim.x, (uint32_t)p.min_share);
    share = (share + kPdWaves - 1) / kPdWaves * kPdWaves;
    uint32_t x = blockIdx.x * share;
    const uint32_t x_end = min(x + share, total);

    while (x < x_end) {   // workgroup-uniform
        // ---- the slab that tile x belongs to ----
        if (s_pre[tid] <= x && x < s_pre[tid + 1]) {
            uint32_t at = s_pre[tid];
            for (int b = b0; b < b1; ++b) {
                Slab s;
                s.len = max(p.c.lens[b], 0);
                keys_of(p, s.len, s.begin, s.end, s.tiles);
                const uint32_t n = (uint32_t)(s.tiles * slabs);
                if (x < at + n) {
                    const uint32_t i = (x - at) / (uint32_t)s.tiles;
                    s.b = b;
                    s.kvh = (int)(i / (uint32_t)p.n_chunks);
                    s.chunk = (int)(i % (uint32_t)p.n_chunks);
                    s.tile0 = s.begin / 32;
                    s.start = at + i * (uint32_t)s.tiles;
                    s_slab = s;
                    break;
                }
                at += n;
            }
        }
        __syncthreads();
        const Slab s = s_slab;
        const int first = (int)(x - s.start);                                    // the piece's tiles [first, last)
        const int last = min(s.tiles, first + (int)(x_end - x));
        const int b = __builtin_amdgcn_readfirstlane(s.b), kvh = __builtin_amdgcn_readfirstlane(s.kvh);
        const int end = __builtin_amdgcn_readfirstlane(s.end), begin = __builtin_amdgcn_readfirstlane(s.begin);
        const int head0 = kvh * p.gqa + s.chunk * p.chunk_heads;
        const int nh = min(p.chunk_heads, p.gqa - s.chunk * p.chunk_heads);
        const int head = head0 + min(c, nh - 1);   // columns past the chunk repeat its last head
        const int pos = s.len - 1;

        u32x4 qb[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            qb[ks] = load16(p.q + ((long)b * p.n_heads + head) * D + 32 * ks + 8 * g);
        const float slope = p.s.slopes ? p.s.slopes[head] * kLog2eF : 0.0f;

        f32x4 o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float m_run = -INFINITY, l_run = 0.0f;   // of column c; l_run: this lane's tokens only

        // This wave's tiles: tile_at(i) = tile0 + first + wave + 4 i, i < count.
        const int base = s.tile0 + first + wave;
        const int count = __builtin_amdgcn_readfirstlane((s.tile0 + last - base + kPdWaves - 1) / kPdWaves);
        const int* table_row = p.c.table + (long)b * p.c.max_pages;
        // Row offsets of 16 tiles ahead: lane l looks up octet l % 4 of the batch's tile l / 4.
        auto look_up = [&](int i0) {
            const int i = i0 + (lane >> 2);
            return i < count ? octet_offset<D>(p.c, table_row, kvh, 32 * (base + kPdWaves * i) + 8 * (lane & 3), end)
                             : -1L;
        };
        long off = look_up(0), off_next = look_up(16);

        auto load = [&](PagedTile<D>& t, int i) {
            const int l0 = 4 * (i & 15);
            const long oz = max(off, 0L);   // an unmapped octet reads the cache's first rows; its tokens are masked
            const int lo = (int)(uint32_t)oz, hi = (int)(oz >> 32);
            if constexpr (UNI) {
                const long row = ((long)__builtin_amdgcn_readlane(hi, l0) << 32) |
                                 (uint32_t)__builtin_amdgcn_readlane(lo, l0);
                const uint16_t* kt = p.c.k + row;
                const uint16_t* vt = p.c.v + row;
#pragma unroll
                for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) t.k[blk][ks] = load16(kt + (uint32_t)((16 * blk + c) * D + 32 * ks + 8 * g));
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint16_t* a = vt + (uint32_t)((16 * (e >> 2) + 4 * g + (e & 3)) * D + VEC * c);
                    if constexpr (VEC == 8) {
                        const u32x4 w = stream16(a);
#pragma unroll
                        for (int i2 = 0; i2 < 4; ++i2) t.v[e][i2] = w[i2];
                    } else {
                        const u32x2 w = stream8(a);
                        t.v[e][0] = w[0];
                        t.v[e][1] = w[1];
                    }
                }
            } else {
                auto row_of = [&](int octet) {
                    return ((long)__shfl(hi, l0 + octet) << 32) | (uint32_t)__shfl(lo, l0 + octet);
                };
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    const uint16_t* kt = p.c.k + row_of(2 * blk + (c >> 3)) + (c & 7) * D + 8 * g;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) t.k[blk][ks] = load16(kt + 32 * ks);
                }
#pragma unroll
                for (int e2 = 0; e2 < 2; ++e2) {
                    const uint16_t* vt = p.c.v + row_of(2 * e2 + (g >> 1)) + 4 * (g & 1) * D + VEC * c;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (VEC == 8) {
                            const u32x4 w = stream16(vt + e * D);
#pragma unroll
                            for (int i2 = 0; i2 < 4; ++i2) t.v[4 * e2 + e][i2] = w[i2];
                        } else {
                            const u32x2 w = stream8(vt + e * D);
                            t.v[4 * e2 + e][0] = w[0];
                            t.v[4 * e2 + e][1] = w[1];
                        }
                    }
                }
            }
        };

        auto step = [&](PagedTile<D>& t, int i, uint64_t unmapped) {
            const int t0 = 32 * (base + kPdWaves * i);
            float sc[8];
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) acc = Hf::mfma16(t.k[blk][ks], qb[ks], acc);
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[4 * blk + r] = acc[r];
            }
            if (p.s.cap_in != 0.0f) {
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
            const uint32_t gone = (uint32_t)(unmapped >> (4 * (i & 15))) & 15u;   // its octets without a page
            if (gone || t0 < begin || t0 + 32 > end) {   // wave-uniform
                // Masked tokens: no score, and no value either (0 * NaN would stay NaN).
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int tok = tk + 16 * (e >> 2) + (e & 3);
                    const bool ok = tok >= begin && tok < end && !((gone >> (2 * (e >> 2) + (g >> 1))) & 1u);
                    if (!ok) {
                        sc[e] = -INFINITY;
#pragma unroll
                        for (int w = 0; w < VW; ++w) t.v[e][w] = 0u;
                    }
                }
            }
            float mx = sc[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sc[e]);
            if (__any(mx > m_run)) {
                mx = fmaxf(xor32_max(xor16_max(mx)), m_run);
                const float a = (m_run == -INFINITY) ? 0.0f : __builtin_amdgcn_exp2f(m_run - mx);
                m_run = mx;
                l_run *= a;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[j][r] *= a;
            }
            const float sub = (m_run == -INFINITY) ? 0.0f : m_run - kPShift;
            u32x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float p0 = __builtin_amdgcn_exp2f(sc[e] - sub), p1 = __builtin_amdgcn_exp2f(sc[e + 1] - sub);
                l_run += p0 + p1;
                const uint32_t h2 = Hf::pack(p0, p1);
                hi[e >> 1] = h2;
                lo[e >> 1] = Hf::pack(p0 - Hf::to_f32((uint16_t)h2), p1 - Hf::to_f32((uint16_t)(h2 >> 16)));
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
                u32x4 a;
#pragma unroll
                for (int i2 = 0; i2 < 4; ++i2) a[i2] = perm_b32(t.v[2 * i2 + 1][j >> 1], t.v[2 * i2][j >> 1], sel);
                o[j] = Hf::mfma16(a, hi, o[j]);
                o[j] = Hf::mfma16(a, lo, o[j]);
            }
        };

        PagedTile<D> ta, tb;
        uint64_t unmapped = __ballot(off < 0);
        if (count > 0) load(ta, 0);
        for (int i = 0; i < count; i += 2) {
            // tile i + 1 never opens a batch of 16 (i is even)
            if (i + 1 < count) load(tb, i + 1);
            step(ta, i, unmapped);
            if (i + 1 >= count) break;
            const uint64_t cur = unmapped;
            if (((i + 2) & 15) == 0) {
                off = off_next;
                unmapped = __ballot(off < 0);
                off_next = look_up(i + 18);
            }
            if (i + 2 < count) load(ta, i + 2);
            step(tb, i + 1, cur);
        }

        // ---- join the waves; write the output or hand the part over ----
        l_run = xor32_sum(xor16_sum(l_run));
        if (c < nh) {
            if (g == 0) {
                s_m[wave][c] = m_run;
                s_l[wave][c] = l_run;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < VEC; j += 4)
                    *reinterpret_cast<f32x4*>(&s_o[wave][c][VEC * (4 * g + r) + j]) =
                        f32x4{o[j][r], o[j + 1][r], o[j + 2][r], o[j + 3][r]};
        }
        __syncthreads();

        const int h = tid >> 4, ch = VEC * (tid & 15);   // this thread's head and channels
        const bool owner = h < nh;
        float wm = -INFINITY, wl = 0.0f, wo[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) wo[e] = 0.0f;
        auto join = [&](float m, float l, const float (&v)[VEC]) {   // a part into (wm, wl, wo)
            const float nm = fmaxf(wm, m);
            if (nm == -INFINITY && l == 0.0f) return;   // (NaN scores leave m = -inf and l = NaN)
            const float a = __builtin_amdgcn_exp2f(wm - nm), w = __builtin_amdgcn_exp2f(m - nm);   // 0 for an empty part
            wl = wl * a + l * w;
#pragma unroll
            for (int e = 0; e < VEC; ++e) wo[e] = wo[e] * a + v[e] * w;
            wm = nm;
        };
        if (owner) {
#pragma unroll
            for (int w = 0; w < kPdWaves; ++w) {
                float v[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] = s_o[w][h][ch + e];
                join(s_m[w][h], s_l[w][h], v);
            }
        }
        const bool whole = first == 0 && last == s.tiles;
        bool finish = whole;
        if (!whole) {
            const uint32_t slot = 2u * blockIdx.x + (first == 0 ? 1u : 0u);
            if (owner) {
                const __amdgpu_buffer_rsrc_t ro =
                    make_buffer_rsrc(p.part_o + (long)slot * p.chunk_heads * D, (uint32_t)(p.chunk_heads * D * 4));
#pragma unroll
                for (int e = 0; e < VEC; e += 4)
                    publish_store16(ro, (uint32_t)(h * D + ch + e) * 4u,
                                    make_u32x4(__float_as_uint(wo[e]), __float_as_uint(wo[e + 1]),
                                               __float_as_uint(wo[e + 2]), __float_as_uint(wo[e + 3])));
                if (ch == 0) {
                    publish_store(&p.part_ml[(slot * p.chunk_heads + h) * 2], wm);
                    publish_store(&p.part_ml[(slot * p.chunk_heads + h) * 2 + 1], wl);
                }
            }
            const uint32_t wg0 = s.start / share, wg1 = (s.start + (uint32_t)s.tiles - 1) / share;
            publish_wait();
            __syncthreads();
            if (tid == 0) s_last = arrive_last(&p.counters[wg0], wg1 - wg0 + 1) ? 1u : 0u;
            __syncthreads();
            finish = s_last != 0;
            if (finish) {
                if (owner) {
                    wm = -INFINITY;
                    wl = 0.0f;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) wo[e] = 0.0f;
                    for (uint32_t w = wg0; w <= wg1; ++w) {
                        const uint32_t sl = 2 * w + (w == wg0 ? 1u : 0u);
                        const __amdgpu_buffer_rsrc_t ro = make_buffer_rsrc(p.part_o + (long)sl * p.chunk_heads * D,
                                                                           (uint32_t)(p.chunk_heads * D * 4));
                        float v[VEC];
#pragma unroll
                        for (int e = 0; e < VEC; e += 4) {
                            const u32x4 r = publish_load16(ro, (uint32_t)(h * D + ch + e) * 4u);
#pragma unroll
                            for (int e2 = 0; e2 < 4; ++e2) {
                                const uint32_t bits = r[e2];
                                v[e + e2] = __uint_as_float(bits);
                            }
                        }
                        join(publish_load(&p.part_ml[(sl * p.chunk_heads + h) * 2]),
                             publish_load(&p.part_ml[(sl * p.chunk_heads + h) * 2 + 1]), v);
                    }
                }
                if (tid == 0) p.counters[wg0] = 0u;   // zero for the next call
            }
        }
        if (finish && owner) {
            if (p.pre_splits) {   // the shared prefix's parts
                const long row = ((long)kvh * p.c.batch + b) * p.gqa + s.chunk * p.chunk_heads + h;
                for (int sp = 0; sp < p.pre_splits; ++sp) {
                    const long at = row * p.pre_splits + sp;
                    float v[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) v[e] = p.pre_o[at * D + ch + e];
                    join(p.pre_ml[2 * at], p.pre_ml[2 * at + 1], v);
                }
            }
            const float inv = wl > 0.0f || wl != wl ? 1.0f / wl : 0.0f;   // a row without keys is zero
            uint16_t* dst = p.out + ((long)b * p.n_heads + head0 + h) * D + ch;
            uint32_t w2[VW];
#pragma unroll
            for (int e = 0; e < VW; ++e) w2[e] = Hf::pack(wo[2 * e] * inv, wo[2 * e + 1] * inv);
            if constexpr (VEC == 8) *reinterpret_cast<u32x4*>(dst) = make_u32x4(w2[0], w2[1], w2[2], w2[3]);
            else *reinterpret_cast<u32x2*>(dst) = u32x2{w2[0], w2[1]};
        }
        x += (uint32_t)(last - first);
        __syncthreads();   // s_slab and the waves' results are read
    }
}

// ---------------------------------------------------------------- host

namespace {

struct PagedDecodePlan {
    int workgroups, chunk_heads, n_chunks, min_share;
    size_t off_o, off_ml, bytes;
};

PagedDecodePlan plan_paged_decode(int batch, int n_heads, int n_kv_heads, int head_dim, long capacity, int cus) {
    PagedDecodePlan pl{};
    const int gqa = n_heads / n_kv_heads;
    pl.n_chunks = (gqa + 15) / 16;
    pl.chunk_heads = (gqa + pl.n_chunks - 1) / pl.n_chunks;
    pl.min_share = 4;
    const long slabs = (long)batch * n_kv_heads * pl.n_chunks;
    const long most = slabs * ((capacity + 31) / 32 / pl.min_share + 1);
    pl.workgroups = (int)std::max(1L, std::min(2L * cus, most));
    const size_t slots = 2 * (size_t)pl.workgroups * pl.chunk_heads;
    pl.off_ml = kCounterBytes;
    pl.off_o = pl.off_ml + align_up(slots * 2 * sizeof(float), 256);
    pl.bytes = pl.off_o + align_up(slots * head_dim * sizeof(float), 256);
    return pl;
}

template <bool BF, int D>
void launch_decode(const PagedDecodeParams& p, int workgroups, bool uniform, hipStream_t stream) {
    if (uniform) paged_decode_kernel<BF, D, true><<<workgroups, kPdThreads, 0, stream>>>(p);
    else paged_decode_kernel<BF, D, false><<<workgroups, kPdThreads, 0, stream>>>(p);
}

}  // namespace

size_t paged_decode_workspace(int batch, int n_heads, int n_kv_heads, int head_dim, long capacity) {
    return plan_paged_decode(batch, n_heads, n_kv_heads, head_dim, capacity, device_cu_count()).bytes;
}

int launch_paged_decode(const PagedLaunch& a, const PagedPrefixParts& pre, hipStream_t stream) {
    const long capacity = std::min((long)a.max_pages * a.page_size, kMaxPagedTokens);
    const PagedDecodePlan pl =
        plan_paged_decode(a.batch, a.n_heads, a.n_kv_heads, a.head_dim, capacity, device_cu_count());
    if (a.workspace == nullptr || a.workspace_bytes < pl.bytes)
        return set_error(LLMIK_ERR_WORKSPACE, "workspace too small (llmik_paged_workspace_size)");
    if ((long)pl.workgroups > kMaxCounters)
        return set_error(LLMIK_ERR_UNSUPPORTED, "too many compute units for the workspace's counters");
    PagedDecodeParams p{};
    p.q = static_cast<const uint16_t*>(a.q);
    p.out = static_cast<uint16_t*>(a.out);
    p.c = paged_view(a);
    p.s = score_opts(a);
    p.n_heads = a.n_heads;
    p.gqa = a.n_heads / a.n_kv_heads;
    p.n_chunks = pl.n_chunks;
    p.chunk_heads = pl.chunk_heads;
    p.first = pre.len;
    p.pre_o = pre.o;
    p.pre_ml = pre.ml;
    p.pre_splits = pre.splits;
    char* ws = static_cast<char*>(a.workspace);
    p.counters = reinterpret_cast<uint32_t*>(ws);
    p.part_ml = reinterpret_cast<float*>(ws + pl.off_ml);
    p.part_o = reinterpret_cast<float*>(ws + pl.off_o);
    p.min_share = pl.min_share;
    const bool uniform = a.page_size % 32 == 0;
    if (a.bf16)
        a.head_dim == 128 ? launch_decode<true, 128>(p, pl.workgroups, uniform, stream)
                          : launch_decode<true, 64>(p, pl.workgroups, uniform, stream);
    else
        a.head_dim == 128 ? launch_decode<false, 128>(p, pl.workgroups, uniform, stream)
                          : launch_decode<false, 64>(p, pl.workgroups, uniform, stream);
    return check_launch();
}

}  // namespace llmik
