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
//      warp 1    : TMEM allocator, tcgen05.mma issuer: O += P V, then S = Q K^T of the stream's next tile (V MN-major, as its pages have it)
//      warps 2-9 : softmax, four warps per stream, one thread per row; P goes back to TMEM as 16-bit pairs, over the scores it came from. O stays in
//                  TMEM and is rescaled only when a row's maximum grows by more than 2^8
//    No causal edge: every row comes behind the whole prefix. (m, l, O) in fp32 go to scratch, one part per split and key stream.
// 2. Own keys, and the end. A CTA has up to 8 query rows of a sequence and KV head; its warps take strips of 16 keys through rings of their
//    own (TMA, three strips ahead, see attention_group.cu, whose arithmetic this is: mma.sync, the weights' rounding kept in the
//    MMA's other 8 rows). Splits of a long sequence are a cluster and meet in its shared memory; there the prefix' parts join, and the rows are
//    written. The scratch has no counters and no state between calls.
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

constexpr int kSpThreads = 320;   // TMA warp + MMA warp + 2 x 4 softmax warps
constexpr int kSpTok = 128;       // keys of a tile, rows of a stream
constexpr int kOwnRows = 8;       // query rows of a CTA of the second part
constexpr int kOwnStrip = 16;     // keys a warp takes at a time; pages hold a multiple
constexpr int kOwnWarps = 4;

struct SharedArgs {
    const void* q;
    void* out;
    int64_t ld_q, ld_out;
    const int32_t* block_tables;
    int max_blocks_per_seq;
    const int4* tiles;      // prefix: (sequence whose table names the pages, first query row, tokens of up to two streams, prefix length)
    const int4* items;      // own keys: pairs (sequence, first query row, tokens, keys), (prefix length, 0, 0, 0)
    int rows, n_q_heads, n_kv_heads, block_size, bs_log2, num_rows_kv;
    int tile_tokens;        // tokens of a stream of rows
    int p_splits, row_tiles;
    int has_prefix;         // the first kernel runs
    float scale_log2;
    float* ws_ml;           // [2 p_splits][rows][n_q_heads][2]; m = -inf: nothing in ws_o
    float* ws_o;            // [2 p_splits][rows][n_q_heads][D]
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
__global__ void __launch_bounds__(kSpThreads, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_kv, const SharedArgs a) {
    constexpr int PANELS = D / 64;
    constexpr int PANEL_BYTES = kSpTok * 128;
    constexpr int TILE_BYTES = PANELS * PANEL_BYTES;
    constexpr int MAX_SLOTS = sp_tiles(D) - 1;
    constexpr uint32_t IDESC_QK = make_idesc_f16(128, kSpTok, kBf16, false, false);
    constexpr uint32_t IDESC_PV = make_idesc_f16(128, D, kBf16, false, true);
    constexpr float kUpLog2 = kBf16 ? 0.0f : 7.0f;     // (2^8 of a stale maximum and these stay below fp16's 2^16)

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + sp_tiles(D) * TILE_BYTES);
    uint64_t* q_full = bars;
    uint64_t* full = bars + 1;
    uint64_t* empty = full + MAX_SLOTS;
    uint64_t* s_full = empty + MAX_SLOTS;    // [stream] S of a tile is there (and P V of the tile before is done)
    uint64_t* p_full = s_full + 2;           // [stream] P is there (and O rescaled)
    uint64_t* o_full = p_full + 2;           // [stream] the last P V is done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
    static_assert((1 + 2 * MAX_SLOTS + 6) * 8 + 4 <= 512, "barriers have room");

    const uint32_t warp = warp_id(), lane = lane_id();
    const int4 tile = a.tiles[blockIdx.x];      // (the plan: no kernel writes it)
    // (in this order: the second kernel, which may start from here on, reads what came before this one without a wait)
    griddep_wait();
    griddep_launch_dependents();
    const int kvh = blockIdx.y, split = blockIdx.z;
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
    // places of K and V of a key tile in the producer's order: K0 K1 V0 K2 V1 ... (two row tiles: K1 is asked for behind K0's products only)
    auto seq_k = [&](int t) { return t < 2 ? t : 2 * t - 1; };
    auto seq_v = [&](int t) { return n_tiles == 1 ? 1 : t >= n_tiles - 1 ? 2 * n_tiles - 1 : 2 * t + 2; };

    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmap_q);
        prefetch_tmap(&tmap_kv);
        mbar_init(q_full, 1);
        for (int i = 0; i < slots; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(&s_full[h], 1);
            mbar_init(&p_full[h], 4);
            mbar_init(&o_full[h], 1);
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

    if (warp == 0) {
        if (lane == 0 && n_tiles > 0) {
            // tile row = token * G + head in group; rows behind the last whole token of 128 are never written, nor stored
            mbar_expect_tx(q_full, (two ? 2 : 1) * PANELS * a.tile_tokens * G * 128);
            for (int q = 0; q < (two ? 2 : 1); ++q)
#pragma unroll
                for (int p = 0; p < PANELS; ++p)
                    tma_load_3d(q_sm + q * TILE_BYTES + p * PANEL_BYTES, &tmap_q, q_full, p * 64, kvh * G, tile.y + q * a.tile_tokens, kEvictFirst);
            const int32_t* table = a.block_tables + static_cast<int64_t>(tile.x) * a.max_blocks_per_seq;
            const int n_blocks = prefix / bs;
            uint32_t slot = 0, phase = 0;
            auto load = [&](int t, int which) {
                mbar_wait(&empty[slot], phase ^ 1);
                uint8_t* dst = ring + slot * TILE_BYTES;
                mbar_expect_tx(&full[slot], TILE_BYTES);
                for (int b = 0; b < bps; ++b) {
                    const int bi = (t0 + t) * bps + b;
                    const int row = bi < n_blocks ? ((table[bi] * 2 + which) * a.n_kv_heads + kvh) * bs : a.num_rows_kv;      // behind the cache: zeros
#pragma unroll
                    for (int p = 0; p < PANELS; ++p) tma_load_2d(dst + p * PANEL_BYTES + b * bs * 128, &tmap_kv, &full[slot], p * 64, row, kEvictNormal);
                }
                if (++slot == static_cast<uint32_t>(slots)) {
                    slot = 0;
                    phase ^= 1;
                }
            };
            load(0, 0);
            if (n_tiles > 1) load(1, 0);
            for (int t = 0; t < n_tiles; ++t) {
                load(t, 1);
                if (t + 2 < n_tiles) load(t + 2, 0);
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && n_tiles > 0) {
            auto wait_full = [&](int seq) { mbar_wait(&full[seq % slots], (seq / slots) & 1); };
            auto issue_qk = [&](int h, int seq) {
                const uint8_t* ktile = ring + (seq % slots) * TILE_BYTES;
                const uint8_t* qtile = q_sm + (two ? h : 0) * TILE_BYTES;
#pragma unroll
                for (int p = 0; p < PANELS; ++p) {
                    const uint64_t dq = make_desc_kmajor_sw128(smem_u32(qtile + p * PANEL_BYTES));
                    const uint64_t dk = make_desc_kmajor_sw128(smem_u32(ktile + p * PANEL_BYTES));
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_f16_ss(tmem_base + h * 128, dq + 2 * k, dk + 2 * k, IDESC_QK, (p > 0 || k > 0) ? 1u : 0u);
                }
                umma_commit(&s_full[h]);
            };
            auto issue_pv = [&](int h, int seq, bool first) {
                const uint8_t* vtile = ring + (seq % slots) * TILE_BYTES;
#pragma unroll
                for (int kk = 0; kk < kSpTok / 16; ++kk)
                    umma_f16_ts(tmem_base + 256 + h * 128, tmem_base + h * 128 + kk * 8,
                                make_desc_mnmajor_sw128(smem_u32(vtile + kk * 16 * 128), PANEL_BYTES), IDESC_PV, (!first || kk > 0) ? 1u : 0u);
            };
            mbar_wait(q_full, 0);
            wait_full(0);
            tc_fence_after();
            issue_qk(0, 0);
            if (two) {
                issue_qk(1, 0);
                umma_commit(&empty[0]);
                for (int t = 0; t < n_tiles; ++t) {
                    const bool more = t + 1 < n_tiles;
                    const int sv = seq_v(t), sk = seq_k(t + 1);
                    if (more) wait_full(sk);
                    wait_full(sv);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        mbar_wait(&p_full[h], t & 1);
                        tc_fence_after();
                        issue_pv(h, sv, t == 0);
                        if (h == 1) umma_commit(&empty[sv % slots]);
                        if (more) issue_qk(h, sk);
                        else umma_commit(&o_full[h]);
                    }
                    if (more) umma_commit(&empty[sk % slots]);
                }
            } else {
                umma_commit(&empty[0]);
                if (n_tiles > 1) {
                    wait_full(1);
                    tc_fence_after();
                    issue_qk(1, 1);
                    umma_commit(&empty[1 % slots]);
                }
                for (int t = 0; t < n_tiles; ++t) {
                    const int h = t & 1, sv = seq_v(t);
                    wait_full(sv);
                    mbar_wait(&p_full[h], (t >> 1) & 1);
                    tc_fence_after();
                    issue_pv(h, sv, t < 2);
                    umma_commit(&empty[sv % slots]);
                    if (t + 2 < n_tiles) {
                        const int sk = seq_k(t + 2);
                        wait_full(sk);
                        tc_fence_after();
                        issue_qk(h, sk);
                        umma_commit(&empty[sk % slots]);
                    } else {
                        umma_commit(&o_full[h]);
                    }
                }
            }
        }
    } else {
        // ===================== softmax / partial output: one thread per row =====================
        const uint32_t quad = warp & 3;              // TMEM lane quadrant this warp may touch
        const int h = (warp - 2) >> 2;               // stream
        const int r = quad * 32 + lane;
        const int row0 = tile.y + (two ? h * a.tile_tokens : 0);
        const int live_rows = (two ? (h == 0 ? a.tile_tokens : tile.z - a.tile_tokens) : tile.z) * G;
        const bool quad_live = static_cast<int>(quad * 32) < live_rows;   // warp-uniform
        const int steps = two ? n_tiles : (n_tiles - h + 1) >> 1;
        const uint32_t tmem_s = tmem_base + h * 128 + ((quad * 32u) << 16);
        const uint32_t tmem_o = tmem_s + 256;
        constexpr float kRescaleThreshold = 8.0f;
        float m_run = -INFINITY, l_run = 0.0f;       // m_run in log2 units, kUpLog2 not in it
        for (int i = 0; i < steps; ++i) {
            mbar_wait(&s_full[h], i & 1);
            tc_fence_after();
            if (!quad_live) {
                if (lane == 0) mbar_arrive(&p_full[h]);
                continue;
            }
            const int left = prefix - (t0 + (two ? i : 2 * i + h)) * kSpTok;      // keys from the tile's first on
            uint32_t sr[128];
#pragma unroll
            for (int c = 0; c < 128; c += 32) tmem_ld_32x32(tmem_s + c, *reinterpret_cast<uint32_t(*)[32]>(&sr[c]));
            tmem_ld_wait();
            if (left < kSpTok) {
#pragma unroll
                for (int j = 0; j < 128; ++j)
                    if (j >= left) sr[j] = __float_as_uint(-INFINITY);
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 128; j += 8)
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
            if (i > 0 && __any_sync(0xffffffffu, grow && !fresh)) {     // (S has arrived: P V of the tile before is done)
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
#pragma unroll
            for (int c = 0; c < 128; c += 64) {
                uint32_t packed[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    float x0, x1;
                    sp_unpack(sp_fma(sp_pack(__uint_as_float(sr[c + 2 * j]), __uint_as_float(sr[c + 2 * j + 1])), k2, m2), x0, x1);
                    x0 = sp_ex2(x0);
                    x1 = sp_ex2(x1);
                    sum[j & 1] = sp_add(sum[j & 1], sp_pack(x0, x1));
                    packed[j] = pack2<kBf16>(x0, x1);
                }
                tmem_st_32x32(tmem_s + c / 2, packed);
            }
            float u0, u1;
            sp_unpack(sp_add(sum[0], sum[1]), u0, u1);
            l_run = l_run * alpha + (u0 + u1);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[h]);
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
            mbar_wait(&o_full[h], 0);
            tc_fence_after();
            if (quad_live) {
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t orr[32];
                    tmem_ld_32x32(tmem_o + c, orr);
                    tmem_ld_wait();
                    if (r < live_rows) {
                        float4* wo = reinterpret_cast<float4*>(a.ws_o + at * D + c);
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            wo[j >> 2] = make_float4(__uint_as_float(orr[j]), __uint_as_float(orr[j + 1]), __uint_as_float(orr[j + 2]), __uint_as_float(orr[j + 3]));
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

// ---- own keys, and the end ---------------------------------------------------------------------------------------------
__host__ __device__ constexpr int own_stages(int d) { return d == 128 ? 3 : 6; }
__host__ __device__ constexpr int own_slot_bytes(int d) { return 2 * kOwnStrip * d * 2; }      // K and V of a strip
__host__ __device__ constexpr int own_smem_bytes(int d) { return kOwnWarps * own_stages(d) * own_slot_bytes(d) + 1024; }

__device__ __forceinline__ uint32_t own_cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void own_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 own_load4(const void* p, uint32_t cta) {
    float4 v;
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [ra];\n\t}\n"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem_u32(p)), "r"(cta) : "memory");
    return v;
}
__device__ __forceinline__ float2 own_load2(const void* p, uint32_t cta) {
    float2 v;
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %2, %3;\n\tld.shared::cluster.v2.f32 {%0, %1}, [ra];\n\t}\n"
                 : "=f"(v.x), "=f"(v.y) : "r"(smem_u32(p)), "r"(cta) : "memory");
    return v;
}

// a running (m, l, four outputs) and one more part of the same row
struct OwnJoin {
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    __device__ __forceinline__ void add(float pm, float pl, const float4& x) {
        if (pm == -INFINITY) return;       // (x may be anything)
        const float mx = fmaxf(m, pm);
        const float w0 = m == -INFINITY ? 0.0f : sp_ex2(m - mx), w1 = sp_ex2(pm - mx);
        l = l * w0 + pl * w1;
        o[0] = o[0] * w0 + x.x * w1;
        o[1] = o[1] * w0 + x.y * w1;
        o[2] = o[2] * w0 + x.z * w1;
        o[3] = o[3] * w0 + x.w * w1;
        m = mx;
    }
};

// grid (splits, items, KV heads * row tiles), splits of an item being a cluster. Lane = 4 * g + t: row g of the MMA is query row g; t picks two of
// every eight keys (as the rows of C and A have it), g the key of K (as the columns of B have it) and, for V, eight output dims.
template <int D, bool kBf16>
__global__ void __launch_bounds__(kOwnWarps * 32, 2)
shared_own_kernel(const __grid_constant__ CUtensorMap tmap_kv, const SharedArgs a) {
    constexpr int W = kOwnWarps;
    constexpr int KC = D / 32;        // 16-byte pieces of a K row per lane
    constexpr int VC = D / 64;        // 16-byte pieces of a V row per lane
    constexpr int LD = D + 4;
    constexpr int ST = own_stages(D);
    constexpr float kUp = kBf16 ? 1.0f : 16384.0f;      // what a weight is multiplied by before it becomes 16 bits
    static_assert(kOwnRows * LD * 4 <= ST * own_slot_bytes(D), "a warp's outputs fit its ring");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[W][ST];
    __shared__ float mg_ml[W][kOwnRows][2];
    __shared__ __align__(16) float cta_o[kOwnRows][D];
    __shared__ __align__(8) float cta_ml[kOwnRows][2];

    // with a prefix the kernel before is ours, and what came before that one is done: only its parts are waited for, below
    if (!a.has_prefix) pdl_enter();
    const int tid = threadIdx.x;
    const int warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int splits = gridDim.x, split = blockIdx.x;
    const int4 item = a.items[2 * blockIdx.y];
    const int prefix = a.items[2 * blockIdx.y + 1].x;
    const int kvh = blockIdx.z / a.row_tiles;
    const int G = a.n_q_heads / a.n_kv_heads;
    const int first_row = (blockIdx.z - kvh * a.row_tiles) * kOwnRows;          // of the item's (token, head) rows
    const int rows = min(item.z * G - first_row, kOwnRows);
    if (rows <= 0) {              // (for the whole cluster)
        if (a.has_prefix) pdl_enter();      // (who waits for this kernel waits for the one before)
        return;
    }
    const int kv_len = item.w;
    const int strips = (kv_len - prefix + kOwnStrip - 1) / kOwnStrip;
    const int per = (strips + splits - 1) / splits;
    const int s0 = split * per + warp, s1 = min(strips, split * per + per);
    if (lane == 0) {
        if (warp == 0) prefetch_tmap(&tmap_kv);
        for (int i = 0; i < ST; ++i) mbar_init(&full[warp][i], 1);
        fence_barrier_init();
    }
    __syncwarp();

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
    const int32_t* table = a.block_tables + static_cast<int64_t>(item.x) * a.max_blocks_per_seq;
    auto first_key = [&](int s) { return prefix + s * kOwnStrip; };
    auto page_of = [&](int s) { return s < s1 ? table[first_key(s) >> a.bs_log2] : 0; };
    uint8_t* ring = smem + warp * ST * own_slot_bytes(D);
    auto load = [&](int s, int blk, int slot) {     // (one lane)
        uint8_t* dst = ring + slot * own_slot_bytes(D);
        const int krow = (((blk * 2) * a.n_kv_heads + kvh) << a.bs_log2) + (first_key(s) & (a.block_size - 1));
        const int vrow = krow + (a.n_kv_heads << a.bs_log2);
        mbar_expect_tx(&full[warp][slot], own_slot_bytes(D));
#pragma unroll
        for (int c = 0; c < VC; ++c) tma_load_2d(dst + c * 2048, &tmap_kv, &full[warp][slot], c * 64, krow, kEvictFirst);
#pragma unroll
        for (int c = 0; c < VC; ++c) tma_load_2d(dst + (VC + c) * 2048, &tmap_kv, &full[warp][slot], c * 64, vrow, kEvictFirst);
    };
    float m_run = -INFINITY, l_run = 0.0f;
    float acc[VC][8][4];
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[c][j][i] = 0.0f;

    int next_page = 0;
    if (lane == 0) {
        int pages[ST];
#pragma unroll
        for (int i = 0; i < ST; ++i) pages[i] = page_of(s0 + i * W);
#pragma unroll
        for (int i = 0; i < ST; ++i)
            if (s0 + i * W < s1) load(s0 + i * W, pages[i], i);
        next_page = page_of(s0 + ST * W);
    }
    int slot = 0;
    uint32_t phase = 0;
    for (int s = s0; s < s1; s += W) {
        const uint8_t* strip = ring + slot * own_slot_bytes(D);
        const int key0 = first_key(s);
        mbar_wait(&full[warp][slot], phase);
        // ---- scores of 16 keys: two chains per tile of 8 ----
        float sc[2][4], sd[2][4];
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
        // ---- weights ----
        float p[4];
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pos = key0 + 2 * t + (i & 1) + 8 * (i >> 1);
            p[i] = live && pos <= q_pos ? (sc[i >> 1][i & 1] + sd[i >> 1][i & 1]) * a.scale_log2 : -INFINITY;
            mx = fmaxf(mx, p[i]);
        }
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
#pragma unroll
        for (int c = 0; c < VC; ++c) {
            uint4 vr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 2 * t + (i & 1) + 8 * (i >> 1);
                vr[i] = *reinterpret_cast<const uint4*>(strip + (VC + c) * 2048 + key * 128 + ((g ^ (key & 7)) << 4));
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
        __syncwarp();       // (the slot has been read)
        if (lane == 0) {
            const int sn = s + ST * W;
            if (sn < s1) load(sn, next_page, slot);
            next_page = page_of(sn + W);
        }
        if (++slot == ST) {
            slot = 0;
            phase ^= 1;
        }
    }

    // ---- the warps' states through shared memory: each in its own ring, whose loads have all been waited for ----
    auto mg_o = [&](int w, int r) { return reinterpret_cast<float*>(smem + w * ST * own_slot_bytes(D)) + r * LD; };
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
    if (live) {
        if (t == 0) {
            mg_ml[warp][g][0] = m_run;
            mg_ml[warp][g][1] = l_run;
        }
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float4* d = reinterpret_cast<float4*>(mg_o(warp, g) + c * 64 + (2 * t + e) * 8);
                auto sum = [&](int j) { return (acc[c][j][e] + acc[c][j][e + 2]) * (1.0f / kUp); };
                d[0] = make_float4(sum(0), sum(1), sum(2), sum(3));
                d[1] = make_float4(sum(4), sum(5), sum(6), sum(7));
            }
    }
    __syncthreads();
    if (a.has_prefix) pdl_enter();
    // the prefix' parts join, and the row is finished
    auto finish = [&](int r, int dd, OwnJoin& j) {
        const int tok = (first_row + r) / G, head = kvh * G + (first_row + r) % G;
        const int64_t row = item.y + tok;
        const int64_t part = static_cast<int64_t>(a.rows) * a.n_q_heads, place = row * a.n_q_heads + head;
        for (int sp = 0; prefix > 0 && sp < 2 * a.p_splits; sp += 8) {        // eight parts' loads at once
            float2 ml[8];
            float4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) ml[i] = sp + i < 2 * a.p_splits ? __ldcg(reinterpret_cast<const float2*>(a.ws_ml + ((sp + i) * part + place) * 2)) : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (ml[i].x != -INFINITY) x[i] = __ldcg(reinterpret_cast<const float4*>(a.ws_o + ((sp + i) * part + place) * D + dd));
#pragma unroll
            for (int i = 0; i < 8; ++i) j.add(ml[i].x, ml[i].y, x[i]);
        }
        uint2 v;
        v.x = pack2<kBf16>(j.o[0] / j.l, j.o[1] / j.l);
        v.y = pack2<kBf16>(j.o[2] / j.l, j.o[3] / j.l);
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + row * a.ld_out + head * D + dd) = v;
    };
    for (int e = tid; e < rows * (D / 4); e += W * 32) {
        const int r = e / (D / 4), dd = (e % (D / 4)) * 4;
        OwnJoin j;
#pragma unroll
        for (int w = 0; w < W; ++w) j.add(mg_ml[w][r][0], mg_ml[w][r][1], *reinterpret_cast<const float4*>(mg_o(w, r) + dd));
        if (splits == 1) {
            finish(r, dd, j);
        } else {
            *reinterpret_cast<float4*>(&cta_o[r][dd]) = make_float4(j.o[0], j.o[1], j.o[2], j.o[3]);
            if (dd == 0) *reinterpret_cast<float2*>(cta_ml[r]) = make_float2(j.m, j.l);
        }
    }
    if (splits == 1) return;
    own_cluster_sync();
    for (int e = tid + static_cast<int>(own_cluster_rank()) * W * 32; e < rows * (D / 4); e += splits * W * 32) {
        const int r = e / (D / 4), dd = (e % (D / 4)) * 4;
        OwnJoin j;
        for (int c = 0; c < splits; ++c) {
            const float2 ml = own_load2(cta_ml[r], c);
            j.add(ml.x, ml.y, own_load4(&cta_o[r][dd], c));
        }
        finish(r, dd, j);
    }
    own_cluster_sync();       // nobody leaves while its sums are read
}

template <int D, bool kBf16>
static int launch_shared(const CUtensorMap& tq, const CUtensorMap& tkv, const CUtensorMap& tstrip, const SharedArgs& a, int n_tiles, int n_items,
                         int o_splits, cudaStream_t s) {
    auto pre = shared_prefix_kernel<D, kBf16>;
    auto own = shared_own_kernel<D, kBf16>;
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        HDS_CHECK_CUDA(cudaFuncSetAttribute(pre, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sp_smem_bytes(D))));
        HDS_CHECK_CUDA(cudaFuncSetAttribute(own, cudaFuncAttributeMaxDynamicSharedMemorySize, own_smem_bytes(D)));
        configured[dev & 63] = true;
    }
    if (n_tiles > 0) HDS_CHECK_CUDA(launch_kernel(pre, dim3(n_tiles, a.n_kv_heads, a.p_splits), dim3(kSpThreads), sp_smem_bytes(D), s, tq, tkv, a));
    HDS_CHECK_CUDA(launch_kernel_cluster(own, o_splits, dim3(o_splits, n_items, a.n_kv_heads * a.row_tiles), dim3(kOwnWarps * 32), own_smem_bytes(D),
                                         s, tstrip, a));
    return HDS_OK;
}

}  // namespace hds

using namespace hds;

extern "C" int64_t hds_paged_attention_shared_workspace_bytes(int rows, int n_q_heads, int head_dim, int p_splits) {
    return static_cast<int64_t>(rows) * n_q_heads * (head_dim + 2) * 4 * 2 * p_splits;
}

extern "C" int hds_paged_attention_shared(const void* q, int64_t ld_q, void* out, int64_t ld_out, int rows, const void* kv_cache_layer,
                                          int64_t num_blocks, const int32_t* block_tables, int max_blocks_per_seq, const int32_t* tiles, int n_tiles,
                                          int p_splits, const int32_t* items, int n_items, int max_tokens, int o_splits, int n_q_heads, int n_kv_heads,
                                          int head_dim, int block_size, float scale, void* workspace, int64_t workspace_bytes, int dtype,
                                          void* stream) {
    HDS_REQUIRE(head_dim == 64 || head_dim == 128, "paged_attention_shared: head_dim must be 64 or 128");
    HDS_REQUIRE(block_size == 16 || block_size == 32 || block_size == 64 || block_size == 128, "paged_attention_shared: block_size must be 16/32/64/128");
    HDS_REQUIRE(n_kv_heads > 0 && n_q_heads > 0 && n_q_heads % n_kv_heads == 0 && n_q_heads / n_kv_heads <= 128,
                "paged_attention_shared: up to 128 query heads per KV head");
    HDS_REQUIRE(dtype == 0 || dtype == 1, "paged_attention_shared: dtype must be 0 (bf16) or 1 (fp16)");
    HDS_REQUIRE(p_splits >= 1 && p_splits <= 64 && (o_splits == 1 || o_splits == 2 || o_splits == 4 || o_splits == 8),
                "paged_attention_shared: 1 to 64 splits of the prefix, 1, 2, 4 or 8 of a sequence's own keys");
    HDS_REQUIRE(n_tiles >= 0 && n_items >= 0 && n_items <= 65535 && rows >= 0 && max_tokens >= 0, "paged_attention_shared: at most 65535 sequences");
    if (n_items == 0 || rows == 0 || max_tokens == 0) return HDS_OK;
    HDS_REQUIRE(ld_q % 8 == 0 && ld_out % 8 == 0 && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
                "paged_attention_shared: rows start on 16-byte boundaries");
    HDS_REQUIRE((reinterpret_cast<uintptr_t>(tiles) & 15) == 0 && (reinterpret_cast<uintptr_t>(items) & 15) == 0, "paged_attention_shared: unaligned work list");
    const int64_t kv_rows = num_blocks * 2 * n_kv_heads * block_size;
    HDS_REQUIRE(num_blocks > 0 && kv_rows < (int64_t(1) << 31), "paged_attention_shared: a layer's cache has fewer than 2^31 page rows");
    const int G = n_q_heads / n_kv_heads;
    SharedArgs a;
    memset(&a, 0, sizeof(a));
    a.row_tiles = static_cast<int>((static_cast<int64_t>(max_tokens) * G + kOwnRows - 1) / kOwnRows);
    HDS_REQUIRE(static_cast<int64_t>(a.row_tiles) * n_kv_heads <= 65535, "paged_attention_shared: too many new tokens in a sequence");
    HDS_REQUIRE(n_tiles == 0 || (workspace != nullptr && workspace_bytes >= hds_paged_attention_shared_workspace_bytes(rows, n_q_heads, head_dim, p_splits) &&
                                 (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                "paged_attention_shared: workspace too small");
    a.q = q; a.out = out; a.ld_q = ld_q; a.ld_out = ld_out;
    a.block_tables = block_tables; a.max_blocks_per_seq = max_blocks_per_seq;
    a.tiles = reinterpret_cast<const int4*>(tiles);
    a.items = reinterpret_cast<const int4*>(items);
    a.rows = rows; a.n_q_heads = n_q_heads; a.n_kv_heads = n_kv_heads;
    a.block_size = block_size;
    a.bs_log2 = block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
    a.num_rows_kv = static_cast<int>(kv_rows);
    a.tile_tokens = 128 / G;
    a.p_splits = p_splits;
    a.has_prefix = n_tiles > 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.ws_o = reinterpret_cast<float*>(workspace);       // the outputs first: they want 16-byte boundaries
    a.ws_ml = a.ws_o + static_cast<int64_t>(2 * p_splits) * rows * n_q_heads * head_dim;
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
    if (head_dim == 128)
        return dtype == 0 ? launch_shared<128, true>(tq, tkv, tstrip, a, n_tiles, n_items, o_splits, s)
                          : launch_shared<128, false>(tq, tkv, tstrip, a, n_tiles, n_items, o_splits, s);
    return dtype == 0 ? launch_shared<64, true>(tq, tkv, tstrip, a, n_tiles, n_items, o_splits, s)
                      : launch_shared<64, false>(tq, tkv, tstrip, a, n_tiles, n_items, o_splits, s);
}
