// Paged attention of a batch whose sequences share a prefix: the prefix' pages are read once for all of them.
//
//   softmax over prefix and own keys = the two parts' (m, l, O) joined:  O = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i
//
// 1. Prefix. All query rows of a group of sequences, (token, query head of the KV head's group) pairs, are rows of one matrix product. A CTA has
//    one KV head, a part of the prefix in tiles of 128 keys, and up to 256 rows: two streams of 128, so that the products of one run while the
//    other one's scores are weighed (the scheme of attention_pair.cuh). With more than 128 rows the streams are two row tiles that see the
//    same keys; with fewer they share the rows and take the key tiles in turn, as two more parts of the prefix.
//      warp 0    : TMA producer - Q (3-D boxes: tokens x heads x 64 dims), then K and V tiles page by page in the order of their use, through one
//                  ring; what is behind the prefix in its last tile comes from behind the cache, that is, as zeros
//      warp 1    : TMEM allocator, tcgen05.mma issuer, for half a tile at a time: O += P V, then S = Q K^T of the same half of the stream's next tile
//                  (V MN-major, as its pages have it)
//      warps 2-9 : softmax, four warps per stream, one thread per row; P goes back to TMEM as 16-bit pairs, over the scores it came from. O stays in
//                  TMEM and is rescaled only when a row's maximum grows by more than 2^8. One half is weighed while the other half's products run:
//                  with products of whole tiles a stream waits for them between two tiles (56.0 us here, 58.4 so at the 65536 keys below; 38.3 and
//                  38.0 at the 8192, where the issue of twice as many products weighs more)
//    No causal edge: every row comes behind the whole prefix. (m, l, O) in fp32 go to scratch, one part per split and key stream.
// 2. Own keys. The warps of a CTA are twelve workers: each takes strips of 16 keys through a ring of its own (TMA, see attention_group.cu, whose
//    arithmetic this is: up to 8 query rows of a sequence and KV head, mma.sync, the weights' rounding kept in the MMA's other 8 rows). All
//    strips of all sequences and heads stand in one line that is cut into pieces of equal cost, one per worker, so that neither long nor short sequences
//    leave SMs idle; a sequence and head costs two strips more than it has, for its beginning and end (with pieces of equal length the worker of the many
//    heads of a short sequence came 25 us behind the others). (m, l, O) of a sequence's share in a piece goes to scratch.
//    These CTAs are of the prefix' launch and begin with it, on so many SMs that both should end together: own keys wait for memory where
//    the prefix waits for its softmax. (One after the other, 4096 shared keys and 32 sequences of 32 heads with 150 keys each took 41.4 us, 64 sequences
//    of 64 heads behind 8192 keys 48.0; together 35.7 and 42.3. Both parts have become faster since.)
// 3. The end: the parts of every row, from prefix and own keys, join in a kernel of their own. The scratch has no counters and no state between calls.
//
// Measured (bf16, bytes that any form has to move, time, bytes per second; a copy runs at 6.55 TB/s):
//   32 sequences, 32 heads of 128 dims and as many KV heads, prefix 4096, 1 to 300 own keys:  147 MB, 32.3 us, 4.6 TB/s
//   64 sequences, 64 heads on 8, prefix 8192, 1 to 600 own keys:                              118 MB, 38.3 us, 3.1 TB/s
//   77 sequences, 32 heads on 8, 1 to 3 new tokens, prefixes 2048 and 1024, 1 to 500 own keys: 93 MB, 30.8 us, 3.0 TB/s
//   9 sequences, 64 heads on 8, prefix 65536, 1 to 1500 own keys:                             294 MB, 56.0 us, 5.3 TB/s
//   4 sequences, 12 heads of 64 dims (fp16), prefix 512, 1 to 90 own keys: 8.7 us, two kernels' beginnings and ends (5 + 3)
// The join and the beginnings are 6 to 8 us of each. Under two row tiles (the second and third line) a key tile takes 2.0 us of a CTA, of which its
// products are 1.1 and its exponentials 1.1: registers and TMEM have room for two streams. Own keys come at 6 TB/s where sequences are long (1200 keys);
// with 150 a worker begins a sequence and head every nine strips. Tokens of which a sequence has two or three have two units of 8 rows, which read the keys
// twice (once from L2).
//
// P is rounded to 16 bits in the first part: each weight by half a step of its own (2^-9 in bf16, 2^-12 in fp16, where the weights are held 2^7
// larger so that small ones keep their bits), which averages out over the keys; sums are of the unrounded weights.
//
// No counterpart in the reference, whose blocked attention (deepspeed/inference/v2/kernels/ragged_ops/blocked_flash/blocked_flash.cpp:21-101)
// reads every sequence's keys for itself.
#include "hds_ptx.cuh"
#include "hds_host.cuh"
#include "mma_sync.cuh"
#include "../../../include/hds_b200.h"

namespace hds {

constexpr int kSpThreads = 384;   // TMA warp + MMA warp + 2 x 4 softmax warps; or 12 workers
constexpr int kSpTok = 128;       // keys of a tile, rows of a stream
constexpr int kOwnRows = 8;       // query rows of a worker
constexpr int kOwnStrip = 16;     // keys a warp takes at a time; pages hold a multiple
constexpr int kOwnWarps = 12;     // workers of a CTA

struct SharedArgs {
    const void* q;
    void* out;
    int64_t ld_q, ld_out;
    const int32_t* block_tables;
    int max_blocks_per_seq;
    const int4* tiles;      // prefix: (sequence whose table names the pages, first query row, tokens of up to two streams, prefix length)
    const int4* items;      // own keys: pairs (sequence, first query row, tokens, keys), (prefix length, first unit, row tiles, 0)
    const int4* workers;    // (item, unit in the item, first strip in the unit, strips)
    const int2* units;      // (first worker, last worker) of a unit: (item, KV head, row tile)
    const int32_t* row_items;   // the item of a query row
    int n_tiles, n_workers, prefix_ctas;
    int rows, n_q_heads, n_kv_heads, block_size, bs_log2, num_rows_kv;
    int tile_tokens;        // tokens of a stream of rows
    int p_splits;
    float scale_log2;
    float* ws_ml;           // [2 p_splits][rows][n_q_heads][2]; m = -inf: nothing in ws_o
    float* ws_o;            // [2 p_splits][rows][n_q_heads][D]
    float* own_ml;          // [units + workers][8][2]: a worker's share of a unit has number unit + worker
    float* own_o;           // [units + workers][8][D]
};

__device__ __forceinline__ float sp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// tiles of 16-bit values in shared memory: Q's one or two, the others a ring of K and V
__host__ __device__ constexpr int sp_tiles(int d) { return d == 128 ? 7 : 13; }
__host__ __device__ constexpr size_t sp_smem_bytes(int d) { return static_cast<size_t>(sp_tiles(d)) * kSpTok * d * 2 + 512 + 1024; }

__device__ __forceinline__ uint64_t sp_pack(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void sp_unpack(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t sp_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t sp_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <int D, bool kBf16>
__device__ __forceinline__ void shared_prefix(const CUtensorMap& tmap_q, const CUtensorMap& tmap_kv, const SharedArgs& a, uint8_t* smem, int block) {
    constexpr int PANELS = D / 64;
    constexpr int PANEL_BYTES = kSpTok * 128;
    constexpr int TILE_BYTES = PANELS * PANEL_BYTES;
    constexpr int MAX_SLOTS = sp_tiles(D) - 1;
    constexpr uint32_t IDESC_QK = make_idesc_f16(128, kSpTok / 2, kBf16, false, false);
    constexpr uint32_t IDESC_PV = make_idesc_f16(128, D, kBf16, false, true);
    constexpr float kUpLog2 = kBf16 ? 0.0f : 7.0f;     // (2^8 of a stale maximum and these stay below fp16's 2^16)

    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + sp_tiles(D) * TILE_BYTES);
    uint64_t* q_full = bars;
    uint64_t* full = bars + 1;
    uint64_t* empty = full + MAX_SLOTS;
    uint64_t* s_full = empty + MAX_SLOTS;    // [stream][half] P V of the tile before is done, and S of half a tile is there unless it was the last one
    uint64_t* p_full = s_full + 4;           // [stream][half] P is there (and O rescaled)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(p_full + 4);
    static_assert((1 + 2 * MAX_SLOTS + 8) * 8 + 4 <= 512, "barriers have room");

    const uint32_t warp = warp_id(), lane = lane_id();
    const int4 tile = a.tiles[block % a.n_tiles];
    const int kvh = block / a.n_tiles % a.n_kv_heads, split = block / a.n_tiles / a.n_kv_heads;
    const int G = a.n_q_heads / a.n_kv_heads;
    const bool two = tile.z > a.tile_tokens;    // two row tiles; else one, whose key tiles the streams share
    const int prefix = tile.w;
    const int tiles_total = (prefix + kSpTok - 1) / kSpTok;
    const int t0 = static_cast<int>(static_cast<int64_t>(tiles_total) * split / a.p_splits);
    const int n_tiles = static_cast<int>(static_cast<int64_t>(tiles_total) * (split + 1) / a.p_splits) - t0;
    const int slots = sp_tiles(D) - (two ? 2 : 1);
    uint8_t* q_sm = smem;                       // [row tile][panel][128 x 64]
    uint8_t* ring = smem + (two ? 2 : 1) * TILE_BYTES;
    const int bs = a.block_size, bps = kSpTok / bs;

    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmap_q);
        prefetch_tmap(&tmap_kv);
        mbar_init(q_full, 1);
        for (int i = 0; i < slots; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc<512>(tmem_slot);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    // The whole warp walks a producer's and an issuer's schedule and one elected lane issues: under `lane == 0` each tcgen05.mma took 90 cycles to
    // issue (64 sequences of 64 heads behind 8192 keys 44.6 us, 39.0 with the elected lane).
    const bool leader = elect_one();
    if (warp == 0) {
        if (n_tiles > 0) {
            // tile row = token * G + head in group; rows behind the last whole token of 128 are never written, nor stored
            if (leader) {
                mbar_expect_tx(q_full, (two ? 2 : 1) * PANELS * a.tile_tokens * G * 128);
                for (int q = 0; q < (two ? 2 : 1); ++q)
#pragma unroll
                    for (int p = 0; p < PANELS; ++p)
                        tma_load_3d(q_sm + q * TILE_BYTES + p * PANEL_BYTES, &tmap_q, q_full, p * 64, kvh * G, tile.y + q * a.tile_tokens, kEvictFirst);
            }
            const int32_t* table = a.block_tables + static_cast<int64_t>(tile.x) * a.max_blocks_per_seq;
            const int n_blocks = prefix / bs;
            uint32_t slot = 0, phase = 0;
            auto load = [&](int t, int which) {
                mbar_wait(&empty[slot], phase ^ 1);
                uint8_t* dst = ring + slot * TILE_BYTES;
                if (leader) mbar_expect_tx(&full[slot], TILE_BYTES);
                for (int b = 0; b < bps; ++b) {
                    const int bi = (t0 + t) * bps + b;
                    const int row = bi < n_blocks ? ((table[bi] * 2 + which) * a.n_kv_heads + kvh) * bs : a.num_rows_kv;      // behind the cache: zeros
                    if (!leader) continue;
#pragma unroll
                    for (int p = 0; p < PANELS; ++p) tma_load_2d(dst + p * PANEL_BYTES + b * bs * 128, &tmap_kv, &full[slot], p * 64, row, kEvictNormal);
                }
                if (++slot == static_cast<uint32_t>(slots)) {
                    slot = 0;
                    phase ^= 1;
                }
            };
            // K0 K1 V0 K2 V1 ... (two row tiles: K1 is asked for behind K0's products only)
            load(0, 0);
            if (n_tiles > 1) load(1, 0);
            for (int t = 0; t < n_tiles; ++t) {
                load(t, 1);
                if (t + 2 < n_tiles) load(t + 2, 0);
            }
        }
    } else if (warp == 1) {
        if (n_tiles > 0) {
            auto commit = [&](uint64_t* bar) {
                if (leader) umma_commit(bar);
            };
            int next = 0;                  // (tiles are used in the order in which they are loaded)
            uint32_t phase = 0;
            auto take = [&]() {            // the slot of the next tile, when it is there
                const int slot = next;
                mbar_wait(&full[slot], phase);
                if (++next == slots) {
                    next = 0;
                    phase ^= 1;
                }
                return slot;
            };
            auto issue_qk = [&](int h, int half, int slot) {
                const uint8_t* ktile = ring + slot * TILE_BYTES + half * (kSpTok / 2) * 128;
                const uint8_t* qtile = q_sm + (two ? h : 0) * TILE_BYTES;
                if (!leader) return;
#pragma unroll
                for (int p = 0; p < PANELS; ++p) {
                    const uint64_t dq = make_desc_kmajor_sw128(smem_u32(qtile + p * PANEL_BYTES));
                    const uint64_t dk = make_desc_kmajor_sw128(smem_u32(ktile + p * PANEL_BYTES));
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_f16_ss(tmem_base + h * 128 + half * 64, dq + 2 * k, dk + 2 * k, IDESC_QK, (p > 0 || k > 0) ? 1u : 0u);
                }
            };
            auto issue_pv = [&](int h, int half, int slot, bool first) {
                const uint64_t dv = make_desc_mnmajor_sw128(smem_u32(ring + slot * TILE_BYTES + half * (kSpTok / 2) * 128), PANEL_BYTES);
                if (!leader) return;
#pragma unroll
                for (int kk = 0; kk < kSpTok / 32; ++kk)        // (16 rows of 128 bytes further: 128 units of 16 bytes)
                    umma_f16_ts(tmem_base + 256 + h * 128, tmem_base + h * 128 + half * 64 + kk * 8, dv + 128 * kk, IDESC_PV, (!first || half > 0 || kk > 0) ? 1u : 0u);
            };
            // P V of half a tile and, if there is a tile behind it for the stream, the products of the same half of that
            auto step = [&](int h, int half, int sv, bool first, uint32_t parity, int sk, bool more) {
                mbar_wait(&p_full[2 * h + half], parity);
                tc_fence_after();
                issue_pv(h, half, sv, first);
                if (more) issue_qk(h, half, sk);
                commit(&s_full[2 * h + half]);
            };
            auto begin = [&](int h, int slot) {
                for (int half = 0; half < 2; ++half) {
                    issue_qk(h, half, slot);
                    commit(&s_full[2 * h + half]);
                }
            };
            mbar_wait(q_full, 0);
            const int k0 = take();
            tc_fence_after();
            begin(0, k0);
            if (two) {
                begin(1, k0);
                commit(&empty[k0]);
                for (int t = 0; t < n_tiles; ++t) {
                    const bool more = t + 1 < n_tiles;
                    const int sk = more ? take() : 0, sv = take();
#pragma unroll 1
                    for (int i = 0; i < 4; ++i) step(i & 1, i >> 1, sv, t == 0, t & 1, sk, more);
                    commit(&empty[sv]);
                    if (more) commit(&empty[sk]);
                }
            } else {
                commit(&empty[k0]);
                if (n_tiles > 1) {
                    const int k1 = take();
                    tc_fence_after();
                    begin(1, k1);
                    commit(&empty[k1]);
                }
                for (int t = 0; t < n_tiles; ++t) {
                    const bool more = t + 2 < n_tiles;
                    const int sv = take(), sk = more ? take() : 0;
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) step(t & 1, half, sv, t < 2, (t >> 1) & 1, sk, more);
                    commit(&empty[sv]);
                    if (more) commit(&empty[sk]);
                }
            }
        }
    } else if (warp < 10) {
        // ===================== softmax / partial output: one thread per row =====================
        const uint32_t quad = warp & 3;              // TMEM lane quadrant this warp may touch
        const int h = (warp - 2) >> 2;               // stream
        const int r = quad * 32 + lane;
        const int row0 = tile.y + (two ? h * a.tile_tokens : 0);
        const int live_rows = (two ? (h == 0 ? a.tile_tokens : tile.z - a.tile_tokens) : tile.z) * G;
        const bool quad_live = static_cast<int>(quad * 32) < live_rows;   // warp-uniform
        const int steps = two ? n_tiles : (n_tiles - h + 1) >> 1;
        const uint32_t tmem_stream = tmem_base + h * 128 + ((quad * 32u) << 16);
        const uint32_t tmem_o = tmem_stream + 256;
        constexpr float kRescaleThreshold = 8.0f;
        float m_run = -INFINITY, l_run = 0.0f;       // m_run in log2 units, kUpLog2 not in it
        for (int i = 0; i < 2 * steps; ++i) {        // half a tile at a time: while one half is weighed, the other one's products run
            const int half = i & 1;
            const uint32_t tmem_s = tmem_stream + half * 64;
            mbar_wait(&s_full[2 * h + half], (i >> 1) & 1);
            tc_fence_after();
            if (!quad_live) {
                if (lane == 0) mbar_arrive(&p_full[2 * h + half]);
                continue;
            }
            const int left = prefix - (t0 + (two ? i >> 1 : (i & ~1) + h)) * kSpTok - half * 64;      // keys from the half's first on
            uint32_t sr[64];
#pragma unroll
            for (int c = 0; c < 64; c += 32) tmem_ld_32x32(tmem_s + c, *reinterpret_cast<uint32_t(*)[32]>(&sr[c]));
            tmem_ld_wait();
            if (left < 64) {
#pragma unroll
                for (int j = 0; j < 64; ++j)
                    if (j >= left) sr[j] = __float_as_uint(-INFINITY);
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 64; j += 8)
#pragma unroll
                for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], fmaxf(__uint_as_float(sr[j + 2 * q]), __uint_as_float(sr[j + 2 * q + 1])));
            const float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            const float m_cand = fmaxf(m_run, tmax * a.scale_log2);
            const bool fresh = (m_run == -INFINITY);
            const bool grow = (m_cand > m_run + kRescaleThreshold) || (fresh && m_cand != -INFINITY);
            const float m_new = grow ? m_cand : m_run;
            const float alpha = (!grow || fresh) ? (grow ? 0.0f : 1.0f) : sp_ex2(m_run - m_new);
            const float m_sub = ((m_new == -INFINITY) ? 0.0f : m_new) - kUpLog2;
            m_run = m_new;
            if (i > 0 && __any_sync(0xffffffffu, grow && !fresh)) {
                mbar_wait(&s_full[2 * h + (half ^ 1)], ((i + 1) >> 1) & 1);     // P V of the half before is done
                tc_fence_after();
                const float f = grow && !fresh ? alpha : 1.0f;
#pragma unroll
                for (int c = 0; c < D; c += 16) {
                    uint32_t orr[16];
                    tmem_ld_32x16(tmem_o + c, orr);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) orr[j] = __float_as_uint(__uint_as_float(orr[j]) * f);
                    tmem_st_32x16(tmem_o + c, orr);
                }
            }
            const uint64_t k2 = sp_pack(a.scale_log2, a.scale_log2), m2 = sp_pack(-m_sub, -m_sub);
            uint64_t sum[2] = {0ull, 0ull};
            uint32_t packed[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                float x0, x1;
                sp_unpack(sp_fma(sp_pack(__uint_as_float(sr[2 * j]), __uint_as_float(sr[2 * j + 1])), k2, m2), x0, x1);
                x0 = sp_ex2(x0);
                x1 = sp_ex2(x1);
                sum[j & 1] = sp_add(sum[j & 1], sp_pack(x0, x1));
                packed[j] = pack2<kBf16>(x0, x1);
            }
            tmem_st_32x32(tmem_s, packed);
            float u0, u1;
            sp_unpack(sp_add(sum[0], sum[1]), u0, u1);
            l_run = l_run * alpha + (u0 + u1);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * h + half]);
        }
        // ---- parts: number `split` and, of the second key stream, p_splits + split (nothing in it with two row tiles) ----
        const int tok = r / G;
        const int64_t place = static_cast<int64_t>(row0 + tok) * a.n_q_heads + kvh * G + (r - tok * G);
        const int64_t part = static_cast<int64_t>(a.rows) * a.n_q_heads;
        const int64_t at = (two ? split : h * a.p_splits + split) * part + place;
        if (r < live_rows) {
            *reinterpret_cast<float2*>(a.ws_ml + at * 2) = make_float2(m_run - kUpLog2, l_run);
            if (two) *reinterpret_cast<float2*>(a.ws_ml + ((a.p_splits + split) * part + place) * 2) = make_float2(-INFINITY, 0.0f);
        }
        if (steps > 0) {
            for (int half = 0; half < 2; ++half) mbar_wait(&s_full[2 * h + half], steps & 1);
            tc_fence_after();
            if (quad_live) {
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t orr[32];
                    tmem_ld_32x32(tmem_o + c, orr);
                    tmem_ld_wait();
                    if (r < live_rows) {
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {       // 32 bytes at a time: whole sectors
                            float v[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(orr[j + e]);
                            st_v8_f32(a.ws_o + at * D + c + j, v);
                        }
                    }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<512>(tmem_base);
    }
}

// ---- own keys ----------------------------------------------------------------------------------------------------------
__host__ __device__ constexpr int own_stages(int d) { return d == 128 ? 2 : 4; }
__host__ __device__ constexpr int own_half_bytes(int d) { return kOwnStrip * d * 2; }      // K or V of a strip
__host__ __device__ constexpr int own_ring_bytes(int d) { return 2 * own_stages(d) * own_half_bytes(d); }
static_assert(kOwnWarps * (own_ring_bytes(128) + 128) <= sp_tiles(128) * kSpTok * 128 * 2 &&
              kOwnWarps * (own_ring_bytes(64) + 128) <= sp_tiles(64) * kSpTok * 64 * 2, "the rings fit");

// Lane = 4 * g + t: row g of the MMA is query row g; t picks two of every eight keys (as the rows of C and A have it), g the key of K (as the
// columns of B have it) and, for V, eight output dims.
template <int D, bool kBf16>
__device__ __forceinline__ void shared_own(const CUtensorMap& tmap_kv, const SharedArgs& a, uint8_t* smem, int worker) {
    constexpr int KC = D / 32;        // 16-byte pieces of a K row per lane
    constexpr int VC = D / 64;        // 16-byte pieces of a V row per lane
    constexpr int ST = own_stages(D);
    constexpr float kUp = kBf16 ? 1.0f : 16384.0f;      // what a weight is multiplied by before it becomes 16 bits
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (warp >= kOwnWarps || worker >= a.n_workers) return;
    uint8_t* ring = smem + warp * own_ring_bytes(D);        // [slot][K, V][panel][16 x 64]
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kOwnWarps * own_ring_bytes(D)) + warp * 2 * ST;        // [slot][K, V]
    if (lane == 0) {
        prefetch_tmap(&tmap_kv);
        for (int i = 0; i < 2 * ST; ++i) mbar_init(&full[i], 1);
        fence_barrier_init();
    }
    __syncwarp();
    const bool leader = elect_one();
    const int G = a.n_q_heads / a.n_kv_heads;
    int n = 0;                           // strips so far: strip n has slot n % ST
    int4 job = a.workers[worker];        // (item, unit in the item, first strip in the unit, strips)
    while (job.w > 0) {
        const int4 item = a.items[2 * job.x], more = a.items[2 * job.x + 1];
        const int prefix = more.x, row_tiles = more.z, kv_len = item.w;
        const int kvh = job.y / row_tiles, first_row = (job.y - kvh * row_tiles) * kOwnRows;       // of the item's (token, head) rows
        const int rows = min(item.z * G - first_row, kOwnRows);
        const int strips = (kv_len - prefix + kOwnStrip - 1) / kOwnStrip;
        const int s0 = job.z, s1 = min(strips, s0 + job.w);
        const int32_t* table = a.block_tables + static_cast<int64_t>(item.x) * a.max_blocks_per_seq;
        auto first_key = [&](int s) { return prefix + s * kOwnStrip; };
        auto page_of = [&](int s) { return s < s1 ? table[first_key(s) >> a.bs_log2] : 0; };
        auto load = [&](int s, int blk, int to, int which) {     // (the elected lane)
            uint8_t* dst = ring + (2 * to + which) * own_half_bytes(D);
            const int row = (((blk * 2 + which) * a.n_kv_heads + kvh) << a.bs_log2) + (first_key(s) & (a.block_size - 1));
            mbar_expect_tx(&full[2 * to + which], own_half_bytes(D));
#pragma unroll
            for (int c = 0; c < VC; ++c) tma_load_2d(dst + c * 2048, &tmap_kv, &full[2 * to + which], c * 64, row, kEvictFirst);
        };
        int v_page = 0, k_page = 0;      // of the strips that V and K are asked for next
        {
            int pages[ST];
#pragma unroll
            for (int i = 0; i < ST; ++i) pages[i] = page_of(s0 + i);
#pragma unroll
            for (int i = 0; i < ST; ++i) {
                if (s0 + i >= s1 || !leader) break;
                load(s0 + i, pages[i], (n + i) % ST, 0);
                load(s0 + i, pages[i], (n + i) % ST, 1);
            }
            v_page = page_of(s0 + ST);
            k_page = page_of(s0 + ST + 1);
        }
        // ---- my query row, pieces of 8 dims permuted as K's are ----
        const bool live = g < rows;
        const int r_tok = live ? (first_row + g) / G : 0, r_head = kvh * G + (live ? (first_row + g) % G : 0);
        const int q_pos = kv_len - item.z + r_tok;
        uint4 q[KC];
        {
            const char* qp = reinterpret_cast<const char*>(a.q) + ((static_cast<int64_t>(item.y) + r_tok) * a.ld_q + r_head * D) * 2 + t * 32;
#pragma unroll
            for (int c = 0; c < KC; ++c)
                q[c] = live ? *reinterpret_cast<const uint4*>(qp + (c >> 1) * 128 + (c & 1) * 16) : make_uint4(0u, 0u, 0u, 0u);
        }
        float m_run = -INFINITY, l_run = 0.0f;
        float acc[VC][8][4];
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[c][j][i] = 0.0f;
        // ---- scores of 16 keys: two chains per tile of 8 ----
        float sc[2][4], sd[2][4];
        auto products = [&](int slot) {
            const uint8_t* strip = ring + 2 * slot * own_half_bytes(D);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[i][e] = sd[i][e] = 0.0f;
            }
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 k = *reinterpret_cast<const uint4*>(strip + (c >> 1) * 2048 + (g + 8 * i) * 128 + (((2 * t + (c & 1)) ^ g) << 4));
                    mma_m16n8k16<kBf16>(sc[i], q[c].x, 0u, q[c].y, 0u, k.x, k.y);
                    mma_m16n8k16<kBf16>(sd[i], q[c].z, 0u, q[c].w, 0u, k.z, k.w);
                }
        };
        mbar_wait(&full[2 * (n % ST)], (n / ST) & 1);
        products(n % ST);
        __syncwarp();
        if (leader && s0 + ST < s1) load(s0 + ST, v_page, n % ST, 0);
        for (int s = s0; s < s1; ++s, ++n) {
            const int slot = n % ST, ahead = (n + 1) % ST;
            const uint8_t* strip = ring + (2 * slot + 1) * own_half_bytes(D);
            const int key0 = first_key(s);
            // ---- weights ----
            float p[4];
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int pos = key0 + 2 * t + (i & 1) + 8 * (i >> 1);
                p[i] = live && pos <= q_pos ? (sc[i >> 1][i & 1] + sd[i >> 1][i & 1]) * a.scale_log2 : -INFINITY;
                mx = fmaxf(mx, p[i]);
            }
            // (the next strip's scores meanwhile; behind the last one a product of anything, which nothing uses)
            if (s + 1 < s1) mbar_wait(&full[2 * ahead], ((n + 1) / ST) & 1);
            products(ahead);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m_run, mx);
            if (__any_sync(0xffffffffu, m_new > m_run)) {
                const float scale = m_run == -INFINITY ? 0.0f : sp_ex2(m_run - m_new);
                l_run *= scale;
#pragma unroll
                for (int c = 0; c < VC; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[c][j][e] *= scale;
                m_run = m_new;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = m_run == -INFINITY ? 0.0f : sp_ex2(p[i] - m_run);
                l_run += p[i];
            }
            // ---- O += P V: rounded weights in rows 0..7, what the rounding left in rows 8..15 ----
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] *= kUp;
            const uint32_t h0 = pack2<kBf16>(p[0], p[1]), h1 = pack2<kBf16>(p[2], p[3]);
            const uint32_t r0 = pack2<kBf16>(p[0] - unpack_lo<kBf16>(h0), p[1] - unpack_hi<kBf16>(h0));
            const uint32_t r1 = pack2<kBf16>(p[2] - unpack_lo<kBf16>(h1), p[3] - unpack_hi<kBf16>(h1));
            mbar_wait(&full[2 * slot + 1], (n / ST) & 1);
#pragma unroll
            for (int c = 0; c < VC; ++c) {
                uint4 vr[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = 2 * t + (i & 1) + 8 * (i >> 1);
                    vr[i] = *reinterpret_cast<const uint4*>(strip + c * 2048 + key * 128 + ((g ^ (key & 7)) << 4));
                    // rows past the last key may hold anything: no weight of zero makes that finite
                    if (key0 + kOwnStrip > kv_len && key0 + key >= kv_len) vr[i] = make_uint4(0u, 0u, 0u, 0u);
                }
                const uint32_t w0[4] = {vr[0].x, vr[0].y, vr[0].z, vr[0].w}, w1[4] = {vr[1].x, vr[1].y, vr[1].z, vr[1].w};
                const uint32_t w2[4] = {vr[2].x, vr[2].y, vr[2].z, vr[2].w}, w3[4] = {vr[3].x, vr[3].y, vr[3].z, vr[3].w};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                    mma_m16n8k16<kBf16>(acc[c][j], h0, r0, h1, r1, __byte_perm(w0[j >> 1], w1[j >> 1], sel), __byte_perm(w2[j >> 1], w3[j >> 1], sel));
                }
            }
            __syncwarp();       // (V of this strip and K of the next one have been read)
            if (leader) {
                if (s + ST < s1) load(s + ST, v_page, slot, 1);
                if (s + ST + 1 < s1) load(s + ST + 1, k_page, ahead, 0);
            }
            v_page = k_page;
            k_page = page_of(s + ST + 2);
        }
        // ---- my share of the unit to scratch ----
        l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
        l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
        if (live) {
            const int64_t at = static_cast<int64_t>(more.y + job.y + worker) * kOwnRows + g;
            if (t == 0) *reinterpret_cast<float2*>(a.own_ml + at * 2) = make_float2(m_run, l_run);
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = (acc[c][j][e] + acc[c][j][e + 2]) * (1.0f / kUp);
                    st_v8_f32(a.own_o + at * D + c * 64 + (2 * t + e) * 8, v);
                }
        }
        // ---- the next unit: of this item, or the first one of the next item that has any ----
        job.w -= s1 - s0;
        job.z = 0;
        if (++job.y == a.n_kv_heads * row_tiles && job.w > 0) {
            job.y = 0;
            do ++job.x;
            while (a.items[2 * job.x + 1].z == 0);
        }
    }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kSpThreads, 1)
shared_parts_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_kv, const __grid_constant__ CUtensorMap tmap_strip,
                    const SharedArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    pdl_enter();
    const int own_ctas = (a.n_workers + kOwnWarps - 1) / kOwnWarps;
    if (static_cast<int>(blockIdx.x) >= own_ctas) shared_prefix<D, kBf16>(tmap_q, tmap_kv, a, smem, blockIdx.x - own_ctas);
    else shared_own<D, kBf16>(tmap_strip, a, smem, blockIdx.x * kOwnWarps + (threadIdx.x >> 5));
}

// ---- the end -------------------------------------------------------------------------------------------------------------
// A row of one head has D / 4 lanes, four outputs each, or `share` times as many where rows are few: then these share out its parts. The lanes of a
// share hold the weights of the parts lane, lane + D / 4, ... of it; then all of them add up the outputs of its parts, eight parts' loads at once.
constexpr int kJoinThreads = 128;

template <int D, bool kBf16>
__global__ void __launch_bounds__(kJoinThreads, 6) shared_join_kernel(const SharedArgs a, int share) {
    constexpr int L = D / 4;
    constexpr int KEEP = 160 / L;          // weights per lane: of 160 parts at a time
    __shared__ float4 other_o[kJoinThreads];
    __shared__ float2 other_ml[kJoinThreads];
    const int lane = threadIdx.x % L, dd = lane * 4, group = threadIdx.x / L, mine = group % share;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * (kJoinThreads / L / share) + group / share;
    const int row = static_cast<int>(min(i / a.n_q_heads, static_cast<int64_t>(a.rows) - 1)), head = static_cast<int>(i % a.n_q_heads);
    const bool in = i < static_cast<int64_t>(a.rows) * a.n_q_heads;
    // (the plan: no kernel writes it)
    const int G = a.n_q_heads / a.n_kv_heads, it = a.row_items[row];
    const int4 item = a.items[2 * it], more = a.items[2 * it + 1];
    const int r = (row - item.y) * G + head % G, unit = more.y + head / G * more.z + r / kOwnRows;
    const int2 workers = a.units[unit];
    const int n_own = workers.y - workers.x + 1, n_pre = more.x > 0 ? 2 * a.p_splits : 0, n = n_pre + n_own;
    const int64_t part = static_cast<int64_t>(a.rows) * a.n_q_heads, place = static_cast<int64_t>(row) * a.n_q_heads + head;
    const int n_mine = (n - mine + share - 1) / share;       // parts mine, mine + share, ...
    auto at = [&](int k) { return k < n_pre ? k * part + place : static_cast<int64_t>(unit + workers.x + k - n_pre) * kOwnRows + r % kOwnRows; };
    pdl_enter();
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    // (all lanes of a warp together, here and below: its rows and shares may have different numbers of parts)
    for (int k0 = 0; __any_sync(0xffffffffu, k0 < n_mine); k0 += KEEP * L) {
        float2 ml[KEEP];
        float mx = m;
#pragma unroll
        for (int q = 0; q < KEEP; ++q) {
            const int j = k0 + q * L + lane, k = mine + j * share;
            ml[q] = j < n_mine ? __ldcg(reinterpret_cast<const float2*>((k < n_pre ? a.ws_ml : a.own_ml) + at(k) * 2)) : make_float2(-INFINITY, 0.0f);
            mx = fmaxf(mx, ml[q].x);
        }
#pragma unroll
        for (int s = L / 2; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
        const float old = m == -INFINITY ? 0.0f : sp_ex2(m - mx);
        l *= old;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= old;
        m = mx;
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < KEEP; ++q) {
            ml[q].x = ml[q].x == -INFINITY ? 0.0f : sp_ex2(ml[q].x - mx);
            sum = fmaf(ml[q].x, ml[q].y, sum);
        }
#pragma unroll
        for (int s = L / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        l += sum;
#pragma unroll
        for (int q = 0; q < KEEP; ++q) {
            const int last = min(n_mine - k0 - q * L, L);
            for (int c = 0; __any_sync(0xffffffffu, c < last); c += 8) {
                float w[8];
                float4 x[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    w[u] = __shfl_sync(0xffffffffu, ml[q].x, (c + u) % L, L);
                    if (c + u >= last) w[u] = 0.0f;
                    const int k = mine + (k0 + q * L + c + u) * share;       // (parts without weight may hold anything)
                    x[u] = w[u] != 0.0f ? __ldcg(reinterpret_cast<const float4*>((k < n_pre ? a.ws_o : a.own_o) + at(k) * D + dd)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    o[0] = fmaf(w[u], x[u].x, o[0]);
                    o[1] = fmaf(w[u], x[u].y, o[1]);
                    o[2] = fmaf(w[u], x[u].z, o[2]);
                    o[3] = fmaf(w[u], x[u].w, o[3]);
                }
            }
        }
    }
    if (share > 1) {
        other_ml[threadIdx.x] = make_float2(m, l);
        other_o[threadIdx.x] = make_float4(o[0], o[1], o[2], o[3]);
        __syncthreads();
        if (mine > 0) return;
        float mx = m;
        for (int k = 1; k < share; ++k) mx = fmaxf(mx, other_ml[threadIdx.x + k * L].x);      // (finite: a row has its own key)
        const float f = sp_ex2(m - mx);
        l *= f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= f;
        for (int k = 1; k < share; ++k) {
            const float2 x = other_ml[threadIdx.x + k * L];
            const float4 y = other_o[threadIdx.x + k * L];
            const float w = sp_ex2(x.x - mx);
            l = fmaf(w, x.y, l);
            o[0] = fmaf(w, y.x, o[0]);
            o[1] = fmaf(w, y.y, o[1]);
            o[2] = fmaf(w, y.z, o[2]);
            o[3] = fmaf(w, y.w, o[3]);
        }
    }
    if (!in) return;
    uint2 v;
    v.x = pack2<kBf16>(o[0] / l, o[1] / l);
    v.y = pack2<kBf16>(o[2] / l, o[3] / l);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + row * a.ld_out + head * D + dd) = v;
}

template <int D, bool kBf16>
static int launch_shared(const CUtensorMap& tq, const CUtensorMap& tkv, const CUtensorMap& tstrip, const SharedArgs& a, cudaStream_t s) {
    auto parts = shared_parts_kernel<D, kBf16>;
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        HDS_CHECK_CUDA(cudaFuncSetAttribute(parts, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sp_smem_bytes(D))));
        configured[dev & 63] = true;
    }
    const int ctas = a.prefix_ctas + (a.n_workers + kOwnWarps - 1) / kOwnWarps;
    HDS_CHECK_CUDA(launch_kernel(parts, dim3(ctas), dim3(kSpThreads), sp_smem_bytes(D), s, tq, tkv, tstrip, a));
    const int64_t threads = static_cast<int64_t>(a.rows) * a.n_q_heads * (D / 4);
    // (as long as all CTAs find room at once: 6 per SM)
    const int room = sm_count() * 6 * kJoinThreads, share = threads <= room / 4 ? 4 : threads <= room / 2 ? 2 : 1;
    HDS_CHECK_CUDA(launch_kernel(shared_join_kernel<D, kBf16>, dim3(static_cast<unsigned>((threads * share + kJoinThreads - 1) / kJoinThreads)), dim3(kJoinThreads), 0,
                                 s, a, share));
    return HDS_OK;
}

}  // namespace hds

using namespace hds;

static int64_t shared_part_floats(int rows, int n_q_heads, int head_dim, int p_splits) {
    return static_cast<int64_t>(rows) * n_q_heads * (head_dim + 2) * 2 * p_splits;
}

extern "C" int64_t hds_paged_attention_shared_workspace_bytes(int rows, int n_q_heads, int head_dim, int n_tiles, int p_splits, int n_units, int n_workers) {
    return 4 * ((n_tiles > 0 ? shared_part_floats(rows, n_q_heads, head_dim, p_splits) : 0) +
                (static_cast<int64_t>(n_units) + n_workers) * kOwnRows * (head_dim + 2));
}

extern "C" int hds_paged_attention_shared(const void* q, int64_t ld_q, void* out, int64_t ld_out, int rows, const void* kv_cache_layer,
                                          int64_t num_blocks, const int32_t* block_tables, int max_blocks_per_seq, const int32_t* tiles, int n_tiles,
                                          int p_splits, const int32_t* items, const int32_t* workers, int n_workers, const int32_t* units, int n_units,
                                          const int32_t* row_items, int n_q_heads, int n_kv_heads, int head_dim, int block_size, float scale,
                                          void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
    HDS_REQUIRE(head_dim == 64 || head_dim == 128, "paged_attention_shared: head_dim must be 64 or 128");
    HDS_REQUIRE(block_size == 16 || block_size == 32 || block_size == 64 || block_size == 128, "paged_attention_shared: block_size must be 16/32/64/128");
    HDS_REQUIRE(n_kv_heads > 0 && n_q_heads > 0 && n_q_heads % n_kv_heads == 0 && n_q_heads / n_kv_heads <= 128,
                "paged_attention_shared: up to 128 query heads per KV head");
    HDS_REQUIRE(dtype == 0 || dtype == 1, "paged_attention_shared: dtype must be 0 (bf16) or 1 (fp16)");
    HDS_REQUIRE(p_splits >= 1 && p_splits <= 64, "paged_attention_shared: 1 to 64 splits of the prefix");
    HDS_REQUIRE(scale >= 0.0f && scale < 0x1p127f, "paged_attention_shared: scale must be below 2^127 and not negative");      // (maxima are of raw scores)
    HDS_REQUIRE(n_tiles >= 0 && rows >= 0 && n_workers >= 0 && n_units >= 0, "paged_attention_shared: negative size");
    if (rows == 0 || n_workers == 0) return HDS_OK;
    HDS_REQUIRE(ld_q % 8 == 0 && ld_out % 8 == 0 && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
                "paged_attention_shared: rows start on 16-byte boundaries");
    HDS_REQUIRE(rows <= 1 || (ld_q >= static_cast<int64_t>(n_q_heads) * head_dim && ld_out >= static_cast<int64_t>(n_q_heads) * head_dim),
                "paged_attention_shared: rows of q or out share memory");
    HDS_REQUIRE(((reinterpret_cast<uintptr_t>(tiles) | reinterpret_cast<uintptr_t>(items) | reinterpret_cast<uintptr_t>(workers)) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(units) & 7) == 0,
                "paged_attention_shared: unaligned work lists");
    const int64_t kv_rows = num_blocks * 2 * n_kv_heads * block_size;
    HDS_REQUIRE(num_blocks > 0 && kv_rows < (int64_t(1) << 31), "paged_attention_shared: a layer's cache has fewer than 2^31 page rows");
    HDS_REQUIRE(static_cast<int64_t>(n_tiles) * n_kv_heads * p_splits < (1 << 30) && static_cast<int64_t>(n_units) + n_workers < (1 << 30) &&
                    static_cast<int64_t>(rows) * n_q_heads * (head_dim / 4) < (int64_t(1) << 38),
                "paged_attention_shared: too much work for one call");
    HDS_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 31) == 0 &&
                    workspace_bytes >= hds_paged_attention_shared_workspace_bytes(rows, n_q_heads, head_dim, n_tiles, p_splits, n_units, n_workers),
                "paged_attention_shared: workspace too small");
    const int G = n_q_heads / n_kv_heads;
    SharedArgs a;
    memset(&a, 0, sizeof(a));
    a.q = q; a.out = out; a.ld_q = ld_q; a.ld_out = ld_out;
    a.block_tables = block_tables; a.max_blocks_per_seq = max_blocks_per_seq;
    a.tiles = reinterpret_cast<const int4*>(tiles);
    a.items = reinterpret_cast<const int4*>(items);
    a.workers = reinterpret_cast<const int4*>(workers);
    a.units = reinterpret_cast<const int2*>(units);
    a.row_items = row_items;
    a.n_tiles = n_tiles; a.n_workers = n_workers; a.prefix_ctas = n_tiles * n_kv_heads * p_splits;
    a.rows = rows; a.n_q_heads = n_q_heads; a.n_kv_heads = n_kv_heads;
    a.block_size = block_size;
    a.bs_log2 = block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
    a.num_rows_kv = static_cast<int>(kv_rows);
    a.tile_tokens = 128 / G;
    a.p_splits = p_splits;
    // Keys that are masked enter as scores of -inf, which are to stay that whatever the scale: a scale of 0 counts as the smallest number above it,
    // which moves no exponent by 2^-20 (scores are below 2^128).
    const float scale_log2 = scale * 1.4426950408889634f;
    a.scale_log2 = scale_log2 > 0.0f ? scale_log2 : 1.401298464e-45f;
    // the outputs first: they want 32-byte boundaries
    const int64_t parts = n_tiles > 0 ? static_cast<int64_t>(2 * p_splits) * rows * n_q_heads : 0;
    const int64_t shares = (static_cast<int64_t>(n_units) + n_workers) * kOwnRows;
    a.ws_o = reinterpret_cast<float*>(workspace);
    a.own_o = a.ws_o + parts * head_dim;
    a.ws_ml = a.own_o + shares * head_dim;
    a.own_ml = a.ws_ml + parts * 2;
    CUtensorMap tq, tkv, tstrip;
    memset(&tq, 0, sizeof(tq));
    int rc;
    if (n_tiles > 0) {
        rc = make_tmap_3d_16b(&tq, q, static_cast<uint64_t>(head_dim), static_cast<uint64_t>(n_q_heads), static_cast<uint64_t>(rows),
                              static_cast<uint64_t>(head_dim) * 2, static_cast<uint64_t>(ld_q) * 2, 64, static_cast<uint32_t>(G),
                              static_cast<uint32_t>(a.tile_tokens), dtype == 0);
        if (rc) return rc;
    }
    rc = make_tmap_2d_16b(&tkv, kv_cache_layer, head_dim, static_cast<uint64_t>(kv_rows), static_cast<uint64_t>(head_dim) * 2, 64, block_size, dtype == 0);
    if (rc) return rc;
    rc = make_tmap_2d_16b(&tstrip, kv_cache_layer, head_dim, static_cast<uint64_t>(kv_rows), static_cast<uint64_t>(head_dim) * 2, 64, kOwnStrip, dtype == 0);
    if (rc) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (head_dim == 128) return dtype == 0 ? launch_shared<128, true>(tq, tkv, tstrip, a, s) : launch_shared<128, false>(tq, tkv, tstrip, a, s);
    return dtype == 0 ? launch_shared<64, true>(tq, tkv, tstrip, a, s) : launch_shared<64, false>(tq, tkv, tstrip, a, s);
}
