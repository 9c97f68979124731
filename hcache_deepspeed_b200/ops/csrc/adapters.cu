// Low-rank adapters of many requests beside a shared projection:  out[t] = base[t] + scale[i] * (x[t] down[i]^T) up[i]^T,  i = ids[t].
//
// Rows are sorted by adapter (the plan's order), and a tile is up to 64 rows of one adapter. Both products run on mma.sync with operands that go
// from memory to registers as the instruction wants them: a sum does not mind its order, so that a lane's 16 bytes of a row are two k-steps'
// worth, and columns of the output are dealt out such that a lane ends up with 8 neighbouring ones, moved 16 bytes at a time.
//
// Few rows (a decode step, tiles of up to 16): one kernel. A cluster of 4 or 8 CTAs has a tile; each sums h = x down^T over its part of the
// width, gives its sums to all of them, over the cluster, and has a part of the outputs. Nothing goes through memory, and what the second
// product reads comes to shared memory while the first one runs.
// Many rows: two kernels. The first sums h over a part of the width for a tile and leaves it in scratch, in fp32; the second has a tile and 256
// outputs. It starts while the first one runs: its part of `up` and of `base` is in registers when h is there.
//
// h enters the second product as a 16-bit value and what its rounding left over, itself in 16 bits, so that it keeps 16 bits or more; fp16
// rows are brought to a largest value of 2^8 ... 2^9 first (and back), since fp16 has no room for large h and few bits for small.
//
// Measured (bytes that any form has to move, time, bytes per second; a copy runs at 6.55 TB/s):
//   1 row, rank 16, 4096 -> 4096: 3.7 us, the chain of one kernel: x and down, a sum over the cluster, up, base
//   64 rows with 61 adapters, rank 16, 4096 -> 11008: 32.8 MB, 10.5 us, 3.1 TB/s: two waves of clusters, each with that chain
//   215 rows of 9 adapters, rank 64, 8192 -> 8192: 29.5 MB, 12.0 us, 2.5 TB/s: the second kernel waits 6 us for h, and needs as long for its one group
//   4099 rows of 6 adapters, rank 32, 4096 -> 4096 (fp16): 103 MB, 36.5 us, 2.8 TB/s: 12 us for x, 24 for base and out, where a group of 64 x 256 outputs
//   takes 0.8 us alone and 3.1 us beside another CTA: loads, stores and fragments through the same pipe, 62% busy, and 16 warps to hide their latency
//
// No counterpart in the reference, whose LoRA linear (deepspeed/linear/optimized_linear.py) has one adapter for all rows.
#include "hds_ptx.cuh"
#include "hds_host.cuh"
#include "mma_sync.cuh"
#include "../../../include/hds_b200.h"

namespace hds {

constexpr int kAdCluster = 8;     // CTAs of a tile in the one kernel, at most
constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kAdMaxRank = 256;
constexpr int kAdRows = 64;       // of a tile
constexpr int kAdFew = 16;        // of a tile that the one kernel takes
constexpr int kAdCols = 256;      // outputs of a CTA of the second of two kernels

struct AdapterArgs {
    const void* x;
    const void* base;
    void* out;
    int ld_x, ld_base, ld_out;
    const void* down;       // [adapters][rank][width]
    const void* up;         // [adapters][outputs][rank]
    const float* scales;    // [adapters]
    const int4* tiles;      // (adapter or -1, place of the first row in the sorted order, rows, 0)
    const int32_t* tile_rows;   // [tiles][64]: the rows, the last one repeated to the end
    int n_adapters, rank, width, outputs, rows;
    int cluster;            // CTAs of a tile: 4 or 8
    int k_parts, k_part;    // parts of the width, and columns of each
    float* h;               // [k_parts][rows][rank], by place in order
};

__device__ __forceinline__ uint32_t ad_cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void ad_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void ad_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// the place of `p` in CTA `cta`'s shared memory
__device__ __forceinline__ uint32_t ad_at(const void* p, uint32_t cta) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(cta));
    return a;
}
__device__ __forceinline__ void ad_store4(uint32_t at, const float4& v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ad_zero() { return make_uint4(0u, 0u, 0u, 0u); }

// h rows of 16-bit values: an odd number of 16 values, so that four rows of a fragment lie in different banks
__host__ __device__ constexpr int ad_pitch(int rank) { return ((rank + 15) / 16 | 1) * 16; }

// (ld: values between rows, below 2^30)
__device__ __forceinline__ const uint16_t* ad_row(const void* p, int row, int ld) {
    return reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(p) + static_cast<int64_t>(row) * (ld * 2));
}

// acc = 16 rows of x times NT * 8 rows of down (those from rb on), over the columns k0 to k1 in blocks of 32, of which this warp has number `b` and
// every `step`-th after it. U of them are asked for at once (rank 16, whole calls of 1 and 64 rows: 3.9 and 10.8 us one by one, 3.7 and 10.6 two,
// 4.1 and 11.0 four). Rows of a tile that are not there repeat others, rows of down behind the rank the last ones: nobody looks at what they come to.
// x1 may be x0.
template <int NT, bool kBf16, int U>
__device__ __forceinline__ void ad_down(float (&acc)[NT][4], const uint16_t* x0, const uint16_t* x1, const uint16_t* down, int rb, int rank, int width, int k0,
                                        int k1, int b, int step, int g, int t) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
    const int last = (rank - rb) / 8 - 1, whole = (k1 - k0) / 32;
    const uint16_t* d0 = down + static_cast<int64_t>(rb + g) * width;
    auto multiply = [&](const uint4& xa, const uint4& xb, const uint4 (&d)[NT]) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            mma_m16n8k16<kBf16>(acc[j], xa.x, xb.x, xa.y, xb.y, d[j].x, d[j].y);
            mma_m16n8k16<kBf16>(acc[j], xa.z, xb.z, xa.w, xb.w, d[j].z, d[j].w);
        }
    };
    for (; b < whole; b += U * step) {
        uint4 xa[U], xb[U], d[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b + u * step < whole) {
                const int k = k0 + (b + u * step) * 32 + t * 8;
                xa[u] = *reinterpret_cast<const uint4*>(x0 + k);
                xb[u] = *reinterpret_cast<const uint4*>(x1 + k);
#pragma unroll
                for (int j = 0; j < NT; ++j) d[u][j] = *reinterpret_cast<const uint4*>(d0 + static_cast<int64_t>(min(j, last) * 8) * width + k);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b + u * step < whole) multiply(xa[u], xb[u], d[u]);
    }
    // a last block of less than 32 columns is the turn of one warp
    if ((k1 - k0) % 32 != 0 && (whole - b) % step == 0) {
        const int k = k0 + whole * 32 + t * 8;
        const bool in = k < k1;
        uint4 d[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) d[j] = in ? *reinterpret_cast<const uint4*>(d0 + static_cast<int64_t>(min(j, last) * 8) * width + k) : ad_zero();
        multiply(in ? *reinterpret_cast<const uint4*>(x0 + k) : ad_zero(), in ? *reinterpret_cast<const uint4*>(x1 + k) : ad_zero(), d);
    }
}

// one row's largest |h| -> the power of two that brings it to 2^8 ... 2^9, and that power's reciprocal, both normal numbers
__device__ __forceinline__ float2 ad_row_scale(float m) {
    const int b = static_cast<int>(__float_as_uint(m) >> 23);               // exponent + 127
    const int e = b == 255 || m == 0.0f ? 0 : min(max(b - 127 - 8, -126), 126);
    return make_float2(__uint_as_float(static_cast<uint32_t>(127 - e) << 23), __uint_as_float(static_cast<uint32_t>(127 + e) << 23));
}
template <bool kBf16>
__device__ __forceinline__ void ad_split(float v, uint16_t& hi, uint16_t& lo) {
    const uint32_t h = pack2<kBf16>(v, 0.0f);
    const float rest = v - unpack_lo<kBf16>(h);
    hi = static_cast<uint16_t>(h);
    lo = static_cast<uint16_t>(pack2<kBf16>(fabsf(rest) < INFINITY ? rest : 0.0f, 0.0f));
}

// 16 rows (r0 and r0 + 8 are this lane's) by 32 outputs from n on. Tile j, column 2 t + e of the MMA is column 8 t + 2 j + e of the 32.
template <bool kBf16>
__device__ __forceinline__ void ad_up_step(float (&acc)[4][4], const uint16_t* h_hi, const uint16_t* h_lo, int pitch, int r0, int c, const uint2 (&u)[4]) {
    const uint2 p0 = *reinterpret_cast<const uint2*>(h_hi + r0 * pitch + c), p1 = *reinterpret_cast<const uint2*>(h_hi + (r0 + 8) * pitch + c);
    const uint2 l0 = *reinterpret_cast<const uint2*>(h_lo + r0 * pitch + c), l1 = *reinterpret_cast<const uint2*>(h_lo + (r0 + 8) * pitch + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        mma_m16n8k16<kBf16>(acc[j], p0.x, p1.x, p0.y, p1.y, u[j].x, u[j].y);
        mma_m16n8k16<kBf16>(acc[j], l0.x, l1.x, l0.y, l1.y, u[j].x, u[j].y);
    }
}
// this lane's values of four rows of `up` (2 j rows on from `up`, which points at its place of a k-step), of which `rows` are left; `in`: the k-step
// has values for this lane
__device__ __forceinline__ void ad_up_load(uint2 (&u)[4], const uint16_t* up, int rank, int rows, bool in) {
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = 2 * j < rows && in ? __ldg(reinterpret_cast<const uint2*>(up + 2 * j * rank)) : make_uint2(0u, 0u);
}
template <bool kBf16>
__device__ __forceinline__ uint4 ad_join(const uint4& b, const float (&acc)[4][4], int e, float s) {
    return make_uint4(pack2<kBf16>(fmaf(s, acc[0][e], unpack_lo<kBf16>(b.x)), fmaf(s, acc[0][e + 1], unpack_hi<kBf16>(b.x))),
                      pack2<kBf16>(fmaf(s, acc[1][e], unpack_lo<kBf16>(b.y)), fmaf(s, acc[1][e + 1], unpack_hi<kBf16>(b.y))),
                      pack2<kBf16>(fmaf(s, acc[2][e], unpack_lo<kBf16>(b.z)), fmaf(s, acc[2][e + 1], unpack_hi<kBf16>(b.z))),
                      pack2<kBf16>(fmaf(s, acc[3][e], unpack_lo<kBf16>(b.w)), fmaf(s, acc[3][e + 1], unpack_hi<kBf16>(b.w))));
}
// rows without an adapter, columns n0 to n1 (multiples of 8)
__device__ __forceinline__ void ad_copy(const AdapterArgs& a, const int4& tile, const int32_t* rows, int n0, int n1) {
    const int pieces = max(0, n1 - n0) / 8;
    for (int i = threadIdx.x; i < tile.z * pieces; i += kAdThreads) {
        const int row = rows[i / pieces], col = n0 + i % pieces * 8;
        *reinterpret_cast<uint4*>(const_cast<uint16_t*>(ad_row(a.out, row, a.ld_out)) + col) = *reinterpret_cast<const uint4*>(ad_row(a.base, row, a.ld_base) + col);
    }
}

// (RANK: of these kernels, or 0 where it is only known when they run: with it addresses are constants and no step is half empty. 64 rows with 61
// adapters, 4096 -> 11008: 13.0 us without and 10.6 with it at rank 16, 18.2 and 14.1 at 32, 43.0 and 36.8 at 64. The powers of two whose sums fit the
// registers in one go have kernels of their own, down to a whole step of the MMA. Others at the same rows: 12.5 us at rank 8, whose steps are half empty,
// 17.8 at 24, 35.4 at 48, and 61 at 128 and 164 at 256, where x is read 2 and 4 times.)

// ---- few rows --------------------------------------------------------------------------------------------------------------
// Each warp has a ring of its own for its groups of 32 rows of `up` (contiguous: one bulk copy each), filled from the start on: 4 groups up to rank
// 16, 2 beyond. Longer rows than 64 values have no room, and go from memory to registers.
constexpr int kAdRingRank = 64;
__host__ __device__ constexpr int ad_ring_slots(int rank) { return rank > kAdRingRank ? 0 : rank <= 16 ? 4 : 2; }
__host__ __device__ constexpr int ad_ring_bytes(int rank) { return ad_ring_slots(rank) * 32 * rank * 2; }
// the sums of the eight CTAs, and before that of the warps; h; its two 16-bit parts
template <int NT>
__host__ __device__ constexpr size_t ad_few_smem_bytes(int rank) {
    const int padded = (rank + NT * 8 - 1) / (NT * 8) * NT * 8;
    return static_cast<size_t>(kAdWarps) * ad_ring_bytes(rank) + (static_cast<size_t>(2 * kAdWarps) * 16 * NT * 8 + 16 * padded) * 4 +
           static_cast<size_t>(2) * 16 * ad_pitch(rank) * 2;
}

template <int NT, int RANK, bool kBf16>
__global__ void __launch_bounds__(kAdThreads, 2) adapter_few_kernel(const AdapterArgs a) {
    constexpr int C = NT * 8;
    extern __shared__ __align__(16) uint8_t ad_smem[];
    __shared__ float row_scale[16];
    __shared__ uint64_t full[kAdWarps][4];
    const int rank = RANK > 0 ? RANK : a.rank, padded = (rank + C - 1) / C * C, pitch = ad_pitch(rank), slots = ad_ring_slots(rank), ctas = a.cluster;
    float* red = reinterpret_cast<float*>(ad_smem + kAdWarps * ad_ring_bytes(rank));      // [8 warps][16][C]
    float* part = red + kAdWarps * 16 * C;                            // [8 CTAs][16][C]
    float* h = part + kAdCluster * 16 * C;                            // [16][padded]
    uint16_t* h_hi = reinterpret_cast<uint16_t*>(h + 16 * padded);    // [16][pitch]
    uint16_t* h_lo = h_hi + 16 * pitch;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    // ---- ahead of the wait for what ran before: the plan, which no kernel writes ----
    griddep_launch_dependents();
    const uint32_t cta = ad_cta_rank();
    const int index = blockIdx.x / ctas;
    const int4 tile = a.tiles[index];
    const int32_t* rows = a.tile_rows + index * kAdRows;
    const int row0 = rows[g], row1 = rows[g + 8];
    const int n_slice = (a.outputs + ctas * 32 - 1) / (ctas * 32) * 32, k_slice = (a.width + ctas * 32 - 1) / (ctas * 32) * 32;
    const int n0 = static_cast<int>(cta) * n_slice, n1 = min(a.outputs, n0 + n_slice);
    const int k0 = static_cast<int>(cta) * k_slice, k1 = min(a.width, k0 + k_slice);
    if (tile.x < 0 || tile.x >= a.n_adapters) {        // (the whole cluster)
        griddep_wait();
        ad_copy(a, tile, rows, n0, n1);
        return;
    }
    const uint16_t* up = reinterpret_cast<const uint16_t*>(a.up) + static_cast<int64_t>(tile.x) * a.outputs * rank;
    const uint16_t* down = reinterpret_cast<const uint16_t*>(a.down) + static_cast<int64_t>(tile.x) * rank * a.width;
    uint8_t* ring = ad_smem + warp * ad_ring_bytes(rank);
    auto load = [&](int n, int slot) {       // (one lane) rows n to n + 31 of `up`, those that are mine
        const uint32_t bytes = static_cast<uint32_t>(min(32, n1 - n)) * rank * 2;
        mbar_expect_tx(&full[warp][slot], bytes);
        bulk_load_1d(ring + slot * 64 * rank, up + static_cast<int64_t>(n) * rank, bytes, &full[warp][slot], kEvictFirst);
    };
    if (lane == 0) {
        for (int i = 0; i < slots; ++i) mbar_init(&full[warp][i], 1);
        fence_barrier_init();
    }
    __syncwarp();
    griddep_wait();
    ad_cluster_arrive();       // (the other CTAs' shared memory may be written from the wait on)
    if (lane == 0)
        for (int i = 0; i < slots; ++i)
            if (n0 + (warp + i * kAdWarps) * 32 < n1) load(n0 + (warp + i * kAdWarps) * 32, i);
    __syncwarp();
    // my two rows of the tile (those that are not there repeat the last one)
    const bool live0 = g < tile.z, live1 = g + 8 < tile.z;
    const uint16_t *x0 = ad_row(a.x, row0, a.ld_x), *x1 = ad_row(a.x, row1, a.ld_x);
    const float scale = a.scales[tile.x];
    const uint16_t *b0 = ad_row(a.base, row0, a.ld_base) + t * 8, *b1 = ad_row(a.base, row1, a.ld_base) + t * 8;
    uint4 next0 = ad_zero(), next1 = ad_zero();       // of base: one group ahead
    auto ask = [&](int n) {
        if (live0 && n + t * 8 < n1) next0 = *reinterpret_cast<const uint4*>(b0 + n);
        if (live1 && n + t * 8 < n1) next1 = *reinterpret_cast<const uint4*>(b1 + n);
    };
    for (int rb = 0; rb < rank; rb += C) {
        // ---- my part of the width, 32 columns at a time, shared out among the warps ----
        float acc[NT][4];
        ad_down<NT, kBf16, NT == 8 ? 1 : 2>(acc, x0, x1, down, rb, rank, a.width, k0, k1, warp, kAdWarps, g, t);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            *reinterpret_cast<float2*>(red + (warp * 16 + g) * C + j * 8 + 2 * t) = make_float2(acc[j][0], acc[j][1]);
            *reinterpret_cast<float2*>(red + (warp * 16 + g + 8) * C + j * 8 + 2 * t) = make_float2(acc[j][2], acc[j][3]);
        }
        if (rb == 0) ask(n0 + warp * 32);
        __syncthreads();
        if (rb == 0) ad_cluster_wait();      // all have begun
        // ---- to everybody, and added up there in the order of the CTAs ----
        for (int i = tid; i < 16 * C / 4; i += kAdThreads) {
            float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kAdWarps; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(red + w * 16 * C + i * 4);
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            for (int p = 0; p < ctas; ++p) ad_store4(ad_at(part + cta * 16 * C + i * 4, p), s);
        }
        ad_cluster_arrive();
        ad_cluster_wait();
        for (int i = tid; i < 16 * C; i += kAdThreads) {
            float s = 0.0f;
            for (int p = 0; p < ctas; ++p) s += part[p * 16 * C + i];
            h[i / C * padded + rb + i % C] = s;
        }
        if (rb + C < rank) {                 // nobody sends the next ones before these are taken
            ad_cluster_arrive();
            ad_cluster_wait();
        }
    }
    __syncthreads();
    if constexpr (!kBf16) {
        for (int r = warp; r < 16; r += kAdWarps) {
            float m = 0.0f;
            for (int c = lane; c < rank; c += 32) m = fmaxf(m, fabsf(h[r * padded + c]));
            m = warp_max(m);
            const float2 f = ad_row_scale(m);
            for (int c = lane; c < rank; c += 32) h[r * padded + c] *= f.x;
            if (lane == 0) row_scale[r] = f.y;
        }
        __syncthreads();
    }
    const int k_steps = (rank + 15) / 16;
    for (int i = tid; i < 16 * k_steps * 16; i += kAdThreads) {
        const int r = i / (k_steps * 16), c = i % (k_steps * 16);
        ad_split<kBf16>(c < rank ? h[r * padded + c] : 0.0f, h_hi[r * pitch + c], h_lo[r * pitch + c]);
    }
    __syncthreads();
    // ---- my part of the outputs, 32 columns at a time ----
    const float s0 = kBf16 ? scale : scale * row_scale[g], s1 = kBf16 ? scale : scale * row_scale[g + 8];
    uint16_t *o0 = const_cast<uint16_t*>(ad_row(a.out, row0, a.ld_out)) + t * 8, *o1 = const_cast<uint16_t*>(ad_row(a.out, row1, a.ld_out)) + t * 8;
    const int first = (g >> 1) * 8 + (g & 1);                 // my row of `up` in a group of 32
    const uint16_t* my_up = up + static_cast<int64_t>(first) * rank + t * 4;
    int slot = 0;
    uint32_t phase = 0;
    for (int n = n0 + warp * 32; n < n1; n += kAdWarps * 32) {
        const bool in = n + t * 8 < n1;
        const uint4 base0 = next0, base1 = next1;
        ask(n + kAdWarps * 32);
        float acc[4][4] = {};
        if (slots > 0) {
            mbar_wait(&full[warp][slot], phase);
            const uint16_t* p = reinterpret_cast<const uint16_t*>(ring + slot * 64 * rank) + first * rank + t * 4;     // (rows that are not there: whatever the slot holds)
            for (int c = 0; c < rank; c += 16) {
                uint2 u[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = c + t * 4 < rank ? *reinterpret_cast<const uint2*>(p + 2 * j * rank + c) : make_uint2(0u, 0u);
                ad_up_step<kBf16>(acc, h_hi, h_lo, pitch, g, c + t * 4, u);
            }
            __syncwarp();       // (the slot has been read)
            if (lane == 0 && n + slots * kAdWarps * 32 < n1) load(n + slots * kAdWarps * 32, slot);
            if (++slot == slots) {
                slot = 0;
                phase ^= 1;
            }
        } else {
            const uint16_t* p = my_up + static_cast<int64_t>(n) * rank;
            for (int c = 0; c < rank; c += 16) {
                uint2 u[4];
                ad_up_load(u, p + c, rank, n1 - n - first, c + t * 4 < rank);
                ad_up_step<kBf16>(acc, h_hi, h_lo, pitch, g, c + t * 4, u);
            }
        }
        if (in && live0) *reinterpret_cast<uint4*>(o0 + n) = ad_join<kBf16>(base0, acc, 0, s0);
        if (in && live1) *reinterpret_cast<uint4*>(o1 + n) = ad_join<kBf16>(base1, acc, 2, s1);
    }
}

// ---- many rows -------------------------------------------------------------------------------------------------------------
// tiles of 16 rows that a tile of so many rows has: 1, 2 or 4, so that they divide the warps
__device__ __forceinline__ int ad_m_tiles(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

__device__ __forceinline__ void ad_copy_async(uint32_t dst, const void* src, bool in) {      // 16 bytes, or zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ad_copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ad_copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A stage holds 64 rows and columns of x (64 x 64, 32 x 128 or 16 x 256 values: 8 KB) and the same columns of NT * 8 rows of down. Every second row
// has the halves of its 128 bytes exchanged, so that the eight 16-byte pieces that a quarter of a warp reads, four of each of two rows, lie in
// different banks.
template <int NT>
__host__ __device__ constexpr int ad_stage_bytes(int m_tiles) { return 8192 + NT * 8 * 512 / m_tiles; }
template <int NT>
__host__ __device__ constexpr int ad_stages(int m_tiles) { return NT == 8 && m_tiles == 1 ? 2 : 4; }     // two CTAs per SM have room
template <int NT>
__host__ __device__ constexpr int ad_down_smem_bytes() { return NT == 8 ? 4 * ad_stage_bytes<NT>(2) : 4 * ad_stage_bytes<NT>(1); }

template <int NT, bool kBf16>
__global__ void __launch_bounds__(kAdThreads, 2) adapter_down_kernel(const AdapterArgs a) {
    constexpr int C = NT * 8;
    extern __shared__ __align__(16) uint8_t ad_smem[];
    float* red = reinterpret_cast<float*>(ad_smem);       // [8 warps][16][C], when the stages have been read
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int4 tile = a.tiles[blockIdx.x];
    const int32_t* rows = a.tile_rows + blockIdx.x * kAdRows;
    const int m_tiles = ad_m_tiles(tile.z), mt = warp % m_tiles, kw = warp / m_tiles, k_warps = kAdWarps / m_tiles;
    const int pieces = 32 / m_tiles, columns = pieces * 8;              // 16-byte pieces and values of a row in a stage
    const int p_log2 = m_tiles == 1 ? 5 : m_tiles == 2 ? 4 : 3;
    const uint16_t* x[2];                                               // my piece of two rows of x per stage
    const int piece = tid & (pieces - 1), first = tid >> p_log2, apart = kAdThreads >> p_log2;
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = ad_row(a.x, rows[first + i * apart], a.ld_x);
    // (in this order: the second kernel, which may start from here on, reads what came before this one without a wait)
    griddep_wait();
    griddep_launch_dependents();
    if (tile.x < 0 || tile.x >= a.n_adapters) return;
    const int k0 = blockIdx.y * a.k_part, k1 = min(a.width, k0 + a.k_part), n_stages = (k1 - k0 + columns - 1) / columns;
    const uint16_t* down = reinterpret_cast<const uint16_t*>(a.down) + static_cast<int64_t>(tile.x) * a.rank * a.width;
    float* h = a.h + (static_cast<int64_t>(blockIdx.y) * a.rows + tile.y) * a.rank;
    const int stage_bytes = ad_stage_bytes<NT>(m_tiles), stages = ad_stages<NT>(m_tiles);
    const uint32_t smem = smem_u32(ad_smem);
    auto place = [&](int row, int p) { return static_cast<uint32_t>((row << p_log2) + (p ^ (row & 1) << 2)) * 16u; };
    for (int rb = 0; rb < a.rank; rb += C) {
        auto load = [&](int s) {        // (always ends a group, an empty one behind the last stage)
            if (s < n_stages) {
                const uint32_t to = smem + (s & (stages - 1)) * stage_bytes;
                const int k = k0 + s * columns + piece * 8;
                const bool in = k < k1;
#pragma unroll
                for (int i = 0; i < 2; ++i) ad_copy_async(to + place(first + i * apart, piece), x[i] + (in ? k : k0), in);
                for (int r = first; r < C; r += apart)
                    ad_copy_async(to + 8192 + place(r, piece), down + static_cast<int64_t>(min(rb + r, a.rank - 1)) * a.width + (in ? k : k0), in);
            }
            ad_copies_end();
        };
        float acc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
        if (rb > 0) __syncthreads();
        for (int s = 0; s < stages - 1; ++s) load(s);
        for (int s = 0; s < n_stages; ++s) {
            if (stages == 4) ad_copies_wait<2>();
            else ad_copies_wait<0>();
            __syncthreads();             // stage s is there, and stage s - 1 has been read
            load(s + stages - 1);
            const uint8_t* from = ad_smem + (s & (stages - 1)) * stage_bytes;
            // blocks of 32 columns: one of this warp's per stage
            const int p = kw * 4 + t;
            const uint4 xa = *reinterpret_cast<const uint4*>(from + place(mt * 16 + g, p)), xb = *reinterpret_cast<const uint4*>(from + place(mt * 16 + g + 8, p));
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const uint4 d = *reinterpret_cast<const uint4*>(from + 8192 + place(j * 8 + g, p));
                mma_m16n8k16<kBf16>(acc[j], xa.x, xb.x, xa.y, xb.y, d.x, d.y);
                mma_m16n8k16<kBf16>(acc[j], xa.z, xb.z, xa.w, xb.w, d.z, d.w);
            }
        }
        ad_copies_wait<0>();
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            *reinterpret_cast<float2*>(red + (warp * 16 + g) * C + j * 8 + 2 * t) = make_float2(acc[j][0], acc[j][1]);
            *reinterpret_cast<float2*>(red + (warp * 16 + g + 8) * C + j * 8 + 2 * t) = make_float2(acc[j][2], acc[j][3]);
        }
        __syncthreads();
        for (int i = tid; i < tile.z * C / 4; i += kAdThreads) {
            const int r = i / (C / 4), c = i % (C / 4) * 4;
            if (rb + c >= a.rank) continue;
            float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int w = 0; w < k_warps; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(red + ((w * m_tiles + (r >> 4)) * 16 + (r & 15)) * C + c);
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            *reinterpret_cast<float4*>(h + static_cast<int64_t>(r) * a.rank + rb + c) = s;
        }
    }
}

// CTA y of a tile has the groups of 256 outputs y, y + gridDim.y, ..., a warp 32 of each. Base goes through a ring in shared memory, all stages of
// which are asked for before h is waited for; `up` goes to registers, KS k-steps of 16 of the next group while this one is computed.
__host__ __device__ constexpr int ad_base_stages(int rank) { return rank <= 32 ? 3 : 2; }      // so that two CTAs fit an SM up to rank 64
__host__ __device__ constexpr int ad_up_smem_bytes(int rank) { return ad_base_stages(rank) * kAdRows * kAdCols * 2 + 2 * kAdRows * ad_pitch(rank) * 2; }

// where 16 bytes of a row of base are: half of the rows have neighbouring four pieces exchanged, as a quarter of a warp reads four of each of two rows
__device__ __forceinline__ int ad_base_piece(int row, int piece) { return piece ^ (row & 1) * 4; }

template <int KS, int RANK, bool kBf16>
__global__ void __launch_bounds__(kAdThreads, 2) adapter_up_kernel(const AdapterArgs a) {
    extern __shared__ __align__(16) uint8_t ad_smem[];
    __shared__ float row_scale[kAdRows];
    __shared__ int rows[kAdRows];
    const int rank = RANK > 0 ? RANK : a.rank, pitch = ad_pitch(rank), k_steps = (rank + 15) / 16, stages = ad_base_stages(rank);
    uint16_t* h_hi = reinterpret_cast<uint16_t*>(ad_smem + stages * kAdRows * kAdCols * 2);            // [64][pitch]
    uint16_t* h_lo = h_hi + kAdRows * pitch;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int4 tile = a.tiles[blockIdx.x];
    const int n_step = gridDim.y * kAdCols, n_first = blockIdx.y * kAdCols;
    if (tile.x < 0 || tile.x >= a.n_adapters) {
        pdl_enter();
        for (int c = n_first; c < a.outputs; c += n_step) ad_copy(a, tile, a.tile_rows + blockIdx.x * kAdRows, c, min(a.outputs, c + kAdCols));
        return;
    }
    // ---- what does not need h: all of it was there before the first kernel let this one start ----
    const int m_tiles = ad_m_tiles(tile.z);
    const uint16_t* up = reinterpret_cast<const uint16_t*>(a.up) + static_cast<int64_t>(tile.x) * a.outputs * rank;
    if (tid < kAdRows) rows[tid] = a.tile_rows[blockIdx.x * kAdRows + tid];
    const float scale = a.scales[tile.x];
    const int first = (g >> 1) * 8 + (g & 1);                 // my row of `up` in a group of 32
    const uint16_t* my_up = up + static_cast<int64_t>(first) * rank + t * 4;
    uint2 next[KS][4];
    auto ask = [&](int at) {        // the first k-steps of `up` for the 32 outputs from `at` on
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) ad_up_load(next[ks], my_up + static_cast<int64_t>(at) * rank + ks * 16, rank, a.outputs - at - first, ks * 16 + t * 4 < rank);
    };
    __syncthreads();
    // a stage: 16 rows per m-tile of 512 bytes; a warp copies a row at a time
    const uint32_t smem = smem_u32(ad_smem);
    auto load = [&](int i) {        // base of group number i (always ends a group of copies, an empty one behind the last)
        const int n = n_first + i * n_step + lane * 8;
        if (n < a.outputs) {
            const uint32_t to = smem + i % stages * (kAdRows * kAdCols * 2) + ad_base_piece(warp, lane) * 16;      // (r is odd where warp is)
            for (int r = warp; r < min(m_tiles * 16, tile.z); r += kAdWarps) ad_copy_async(to + r * kAdCols * 2, ad_row(a.base, rows[r], a.ld_base) + n, true);
        }
        ad_copies_end();
    };
    for (int i = 0; i < stages; ++i) load(i);
    ask(n_first + warp * 32);
    griddep_wait();
    griddep_launch_dependents();
    // ---- h, summed over the parts of the width, in two 16-bit values: a row has a power of two of lanes, four values each at a time ----
    const float* h = a.h + static_cast<int64_t>(tile.y) * rank;
    const int64_t part = static_cast<int64_t>(a.rows) * rank;
    const int lanes = rank <= 16 ? 4 : rank <= 32 ? 8 : rank <= 64 ? 16 : 32, per_warp = 32 / lanes, c0 = (lane & (lanes - 1)) * 4;
    for (int r = warp * per_warp + lane / lanes; r < m_tiles * 16; r += kAdWarps * per_warp) {
        float4 s[kAdMaxRank / 128];
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < kAdMaxRank / 128; ++i) {
            s[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const int c = c0 + i * 128;
            if (r < tile.z && c < rank)
                for (int p = 0; p < a.k_parts; ++p) {
                    const float4 v = __ldcg(reinterpret_cast<const float4*>(h + p * part + r * rank + c));
                    s[i].x += v.x; s[i].y += v.y; s[i].z += v.z; s[i].w += v.w;
                }
            m = fmaxf(m, fmaxf(fmaxf(fabsf(s[i].x), fabsf(s[i].y)), fmaxf(fabsf(s[i].z), fabsf(s[i].w))));
        }
        float2 f = make_float2(1.0f, 1.0f);
        if constexpr (!kBf16) {
            for (int o = lanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            f = ad_row_scale(m);
            if (c0 == 0) row_scale[r] = f.y;
        }
#pragma unroll
        for (int i = 0; i < kAdMaxRank / 128; ++i) {
            const int c = c0 + i * 128;
            if (c >= k_steps * 16) continue;
            s[i].x *= f.x; s[i].y *= f.x; s[i].z *= f.x; s[i].w *= f.x;
            const uint2 hi = make_uint2(pack2<kBf16>(s[i].x, s[i].y), pack2<kBf16>(s[i].z, s[i].w));
            auto rest = [](float v, float of) { const float d = v - of; return fabsf(d) < INFINITY ? d : 0.0f; };
            *reinterpret_cast<uint2*>(h_hi + r * pitch + c) = hi;
            *reinterpret_cast<uint2*>(h_lo + r * pitch + c) =
                make_uint2(pack2<kBf16>(rest(s[i].x, unpack_lo<kBf16>(hi.x)), rest(s[i].y, unpack_hi<kBf16>(hi.x))),
                           pack2<kBf16>(rest(s[i].z, unpack_lo<kBf16>(hi.y)), rest(s[i].w, unpack_hi<kBf16>(hi.y))));
        }
    }
    int row[kAdRows / 16][2];
#pragma unroll
    for (int m = 0; m < kAdRows / 16; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) row[m][e] = rows[m * 16 + g + 8 * e];
    for (int i = 0, n0 = n_first; n0 < a.outputs; ++i, n0 += n_step) {
        const int n = n0 + warp * 32, col = n + t * 8;        // (a warp whose 32 are behind the end writes nothing)
        uint2 u[KS][4];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int q = 0; q < 4; ++q) u[ks][q] = next[ks][q];
        ask(n + n_step);
        if (stages == 3) ad_copies_wait<2>();
        else ad_copies_wait<1>();
        __syncthreads();            // the stage is there, and h
        uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + col;
        const uint8_t* base = ad_smem + i % stages * (kAdRows * kAdCols * 2) + ad_base_piece(g, warp * 4 + t) * 16;
#pragma unroll
        for (int m = 0; m < kAdRows / 16; ++m) {
            if (m >= m_tiles) break;
            const int r0 = m * 16 + g;
            float acc[4][4] = {};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                if (ks < k_steps) ad_up_step<kBf16>(acc, h_hi, h_lo, pitch, r0, ks * 16 + t * 4, u[ks]);
            for (int ks = KS; ks < k_steps; ++ks) {
                uint2 more[4];
                ad_up_load(more, my_up + static_cast<int64_t>(n) * rank + ks * 16, rank, a.outputs - n - first, ks * 16 + t * 4 < rank);
                ad_up_step<kBf16>(acc, h_hi, h_lo, pitch, r0, ks * 16 + t * 4, more);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (col < a.outputs && r0 + 8 * e < tile.z)
                    *reinterpret_cast<uint4*>(const_cast<uint16_t*>(ad_row(out, row[m][e], a.ld_out))) =
                        ad_join<kBf16>(*reinterpret_cast<const uint4*>(base + (r0 + 8 * e) * kAdCols * 2), acc, 2 * e, kBf16 ? scale : scale * row_scale[r0 + 8 * e]);
        }
        __syncthreads();            // the stage has been read
        load(i + stages);
    }
    ad_copies_wait<0>();
}

template <int NT, int RANK, bool kBf16>
static int launch_few(const AdapterArgs& a, int n_tiles, cudaStream_t s) {
    auto kern = adapter_few_kernel<NT, RANK, kBf16>;
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        HDS_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(ad_few_smem_bytes<NT>(NT == 2 ? 16 : NT == 4 ? 32 : kAdRingRank) > ad_few_smem_bytes<NT>(kAdMaxRank)
                                                                  ? ad_few_smem_bytes<NT>(NT == 2 ? 16 : NT == 4 ? 32 : kAdRingRank)
                                                                  : ad_few_smem_bytes<NT>(kAdMaxRank))));
        configured[dev & 63] = true;
    }
    HDS_CHECK_CUDA(launch_kernel_cluster(kern, a.cluster, dim3(static_cast<unsigned>(n_tiles) * a.cluster), dim3(kAdThreads),
                                         ad_few_smem_bytes<NT>(a.rank), s, a));
    return HDS_OK;
}

template <int NT, int KS, int RANK, bool kBf16>
static int launch_many(const AdapterArgs& a, int n_tiles, cudaStream_t s) {
    auto down = adapter_down_kernel<NT, kBf16>;
    auto up = adapter_up_kernel<KS, RANK, kBf16>;
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        HDS_CHECK_CUDA(cudaFuncSetAttribute(down, cudaFuncAttributeMaxDynamicSharedMemorySize, ad_down_smem_bytes<NT>()));
        HDS_CHECK_CUDA(cudaFuncSetAttribute(up, cudaFuncAttributeMaxDynamicSharedMemorySize, ad_up_smem_bytes(KS == 1 ? 16 : KS == 2 ? 32 : kAdMaxRank)));
        configured[dev & 63] = true;
    }
    HDS_CHECK_CUDA(launch_kernel(down, dim3(n_tiles, a.k_parts), dim3(kAdThreads), ad_down_smem_bytes<NT>(), s, a));
    // CTAs of a tile: the fewest waves of two per SM, a CTA's beginning and end counted as one group of outputs
    const int groups = (a.outputs + kAdCols - 1) / kAdCols, slots = 2 * sm_count();
    int parts = 1;
    int64_t best = INT64_MAX;
    for (int p = 1; p <= groups; ++p) {
        const int64_t cost = (static_cast<int64_t>(n_tiles) * p + slots - 1) / slots * ((groups + p - 1) / p + 1);
        if (cost < best) {
            best = cost;
            parts = p;
        }
        if (static_cast<int64_t>(n_tiles) * p >= slots && p >= 8) break;
    }
    HDS_CHECK_CUDA(launch_kernel(up, dim3(n_tiles, parts), dim3(kAdThreads), ad_up_smem_bytes(a.rank), s, a));
    return HDS_OK;
}

template <int NT, int RANK, bool kBf16>
static int launch_adapters_as(const AdapterArgs& a, int n_tiles, bool few, cudaStream_t s) {
    return few ? launch_few<NT, RANK, kBf16>(a, n_tiles, s) : launch_many<NT, NT / 2, RANK, kBf16>(a, n_tiles, s);
}
template <bool kBf16>
static int launch_adapters(const AdapterArgs& a, int n_tiles, bool few, cudaStream_t s) {
    if (a.rank == 16) return launch_adapters_as<2, 16, kBf16>(a, n_tiles, few, s);
    if (a.rank == 32) return launch_adapters_as<4, 32, kBf16>(a, n_tiles, few, s);
    if (a.rank == 64) return launch_adapters_as<8, 64, kBf16>(a, n_tiles, few, s);
    return a.rank < 16 ? launch_adapters_as<2, 0, kBf16>(a, n_tiles, few, s)
           : a.rank < 32 ? launch_adapters_as<4, 0, kBf16>(a, n_tiles, few, s) : launch_adapters_as<8, 0, kBf16>(a, n_tiles, few, s);
}

}  // namespace hds

using namespace hds;

// Parts of the width of the first of two kernels: two CTAs on every SM, of at least 256 columns each, and no more than 16, which the second one adds
// up (215 rows of 9 adapters, rank 64, 8192 -> 8192: 12.0 us with 16, 12.5 with 32, 14.4 with 8).
extern "C" int hds_adapter_parts(int n_tiles, int width) {
    const int most = (width + 255) / 256;
    int parts = n_tiles > 0 ? (2 * sm_count() + n_tiles / 2) / n_tiles : 1;
    parts = parts < 1 ? 1 : parts > most ? most : parts;
    return parts > 16 ? 16 : parts;
}

extern "C" int hds_adapter_add(const void* base, int64_t ld_base, const void* x, int64_t ld_x, const void* down, const void* up, const float* scales,
                               int n_adapters, int rank, int width, int outputs, int rows, const int32_t* tiles, const int32_t* tile_rows, int n_tiles,
                               int most_rows, void* out, int64_t ld_out, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
    HDS_REQUIRE(dtype == 0 || dtype == 1, "adapter_add: dtype must be 0 (bf16) or 1 (fp16)");
    HDS_REQUIRE(rank >= 8 && rank <= kAdMaxRank && rank % 8 == 0, "adapter_add: ranks are multiples of 8 up to 256");
    HDS_REQUIRE(width > 0 && outputs > 0 && width % 8 == 0 && outputs % 8 == 0 && width < (1 << 24) && outputs < (1 << 24),
                "adapter_add: widths are multiples of 8 below 2^24");
    HDS_REQUIRE(ld_base % 8 == 0 && ld_x % 8 == 0 && ld_out % 8 == 0, "adapter_add: rows start on 16-byte boundaries");
    HDS_REQUIRE(ld_base >= 0 && ld_x >= 0 && ld_out >= 0 && ld_base < (1 << 30) && ld_x < (1 << 30) && ld_out < (1 << 30), "adapter_add: rows are less than 2^30 apart");
    HDS_REQUIRE(rows <= 1 || ld_out >= outputs, "adapter_add: rows of out share memory");
    HDS_REQUIRE(((reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(down) |
                  reinterpret_cast<uintptr_t>(up) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(tiles)) & 15) == 0,
                "adapter_add: operands start on 16-byte boundaries");
    HDS_REQUIRE(most_rows >= 0 && most_rows <= kAdRows, "adapter_add: tiles of up to 64 rows");
    HDS_REQUIRE(n_tiles >= 0 && n_tiles <= (1 << 26) && rows >= 0, "adapter_add: too many tiles");
    if (n_tiles == 0) return HDS_OK;
    AdapterArgs a;
    memset(&a, 0, sizeof(a));
    a.x = x; a.base = base; a.out = out;
    a.ld_x = static_cast<int>(ld_x); a.ld_base = static_cast<int>(ld_base); a.ld_out = static_cast<int>(ld_out);
    a.down = down; a.up = up; a.scales = scales; a.tiles = reinterpret_cast<const int4*>(tiles); a.tile_rows = tile_rows;
    a.n_adapters = n_adapters; a.rank = rank; a.width = width; a.outputs = outputs; a.rows = rows;
    const bool few = workspace == nullptr;
    HDS_REQUIRE(!few || most_rows <= kAdFew, "adapter_add: tiles of more than 16 rows need a workspace");
    a.cluster = n_tiles * 8 <= sm_count() ? 8 : 4;
    if (!few) {
        const int parts = hds_adapter_parts(n_tiles, width);
        a.k_part = ((width + parts - 1) / parts + 31) / 32 * 32;
        a.k_parts = (width + a.k_part - 1) / a.k_part;
        HDS_REQUIRE(workspace_bytes >= static_cast<int64_t>(parts) * rows * rank * 4 && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
                    "adapter_add: workspace too small");
        a.h = static_cast<float*>(workspace);
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == 0 ? launch_adapters<true>(a, n_tiles, few, s) : launch_adapters<false>(a, n_tiles, few, s);
}
