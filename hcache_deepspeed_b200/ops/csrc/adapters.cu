// Low-rank adapters of many requests beside a shared projection:  out[t] = base[t] + scale[i] * (x[t] down[i]^T) up[i]^T,  i = ids[t].
//
// Rows are sorted by adapter (the plan's order), and a tile is up to 16 or 64 rows of one adapter. A cluster of 8 CTAs has a tile:
//   1. h = x down^T: CTA r sums over its eighth of the width. Both operands go from memory to registers as mma.sync wants them (a sum
//      does not mind its order, so a lane's 16 bytes of a row are two k-steps' worth).
//   2. The eighths meet in shared memory, over the cluster: CTA r adds up the eighth r of the tile's h (in the order of the CTAs) and gives
//      the sums to all of them. No scratch in global memory, no tickets: calls on several streams and captured graphs share nothing.
//   3. out = base + scale h up^T: CTA r has an eighth of the outputs, in groups of 32 columns whose order in the MMA is such that a
//      lane ends up with 8 neighbouring ones: base and out are moved 16 bytes at a time.
// h enters the second product as a 16-bit value and what its rounding left over, itself in 16 bits, so that it keeps 16 bits or more; fp16
// rows are brought to a largest value of 2^8 ... 2^9 first (and back), since fp16 has no room for large h and few bits for small.
//
// No counterpart in the reference, whose LoRA linear (deepspeed/linear/optimized_linear.py) has one adapter for all rows.
#include "hds_ptx.cuh"
#include "hds_host.cuh"
#include "mma_sync.cuh"
#include "../../../include/hds_b200.h"

namespace hds {

constexpr int kAdCluster = 8;
constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kAdMaxRank = 256;

struct AdapterArgs {
    const void* x;
    const void* base;
    void* out;
    int64_t ld_x, ld_base, ld_out;
    const void* down;       // [adapters][rank][width]
    const void* up;         // [adapters][outputs][rank]
    const float* scales;    // [adapters]
    const int32_t* order;   // rows sorted by adapter
    const int4* tiles;      // (adapter or -1, first place in order, rows, 0)
    int n_adapters, rank, width, outputs;
};

__device__ __forceinline__ uint32_t ad_cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void ad_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the place of `p` in CTA `cta`'s shared memory
__device__ __forceinline__ uint32_t ad_at(const void* p, uint32_t cta) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(cta));
    return a;
}
__device__ __forceinline__ float4 ad_load4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void ad_store4(uint32_t at, const float4& v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ad_zero() { return make_uint4(0u, 0u, 0u, 0u); }

template <int MT>
__host__ __device__ constexpr int ad_rows() { return 16 * MT; }
// h rows of 16-bit values: 8 more than the rank, so that the rows of a fragment lie in different banks
__host__ __device__ constexpr int ad_pitch(int rank) { return (rank + 15) / 16 * 16 + 8; }
// the warps' sums of a block of 64 of the rank, then those of the CTA and of all CTAs, then the two 16-bit parts of h
template <int MT>
__host__ __device__ constexpr size_t ad_smem_bytes(int rank) {
    const int padded = (rank + 63) / 64 * 64;
    return (static_cast<size_t>(kAdWarps) * 16 * 64 + ad_rows<MT>() * 64 + static_cast<size_t>(ad_rows<MT>()) * padded) * 4 +
           static_cast<size_t>(2) * ad_rows<MT>() * ad_pitch(rank) * 2;
}

template <int MT, int NT, bool kBf16>
__global__ void __launch_bounds__(kAdThreads) adapter_kernel(const AdapterArgs a) {
    constexpr int M = ad_rows<MT>();
    constexpr int KW = kAdWarps / MT;           // warps that share a tile of 16 rows
    extern __shared__ __align__(16) uint8_t ad_smem[];
    __shared__ float row_scale[M];
    const int rank = a.rank, padded = (rank + 63) / 64 * 64, pitch = ad_pitch(rank);
    float* red = reinterpret_cast<float*>(ad_smem);                   // [8 warps][16][64]
    float* part = red + kAdWarps * 16 * 64;                           // [M][64]
    float* h = part + M * 64;                                         // [M][padded]
    uint16_t* h_hi = reinterpret_cast<uint16_t*>(h + M * padded);     // [M][pitch]
    uint16_t* h_lo = h_hi + M * pitch;
    pdl_enter();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t cta = ad_cta_rank();
    const int4 tile = a.tiles[blockIdx.x / kAdCluster];
    const int n_slice = (a.outputs + kAdCluster * 32 - 1) / (kAdCluster * 32) * 32;
    const int n0 = static_cast<int>(cta) * n_slice, n1 = min(a.outputs, n0 + n_slice);
    if (tile.x < 0 || tile.x >= a.n_adapters) {        // rows without an adapter (the whole cluster leaves here)
        const int pieces = max(0, n1 - n0) / 8;
        for (int i = tid; i < tile.z * pieces; i += kAdThreads) {
            const int64_t row = a.order[tile.y + i / pieces];
            const int64_t col = n0 + i % pieces * 8;
            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + row * a.ld_out + col) =
                *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.base) + row * a.ld_base + col);
        }
        return;
    }
    const int mt = warp % MT, kw = warp / MT;
    const int r0 = mt * 16 + g, r1 = r0 + 8;           // my two rows of the tile
    const bool live0 = r0 < tile.z, live1 = r1 < tile.z;
    const int64_t row0 = a.order[tile.y + (live0 ? r0 : 0)], row1 = a.order[tile.y + (live1 ? r1 : 0)];
    const uint16_t* x0 = reinterpret_cast<const uint16_t*>(a.x) + row0 * a.ld_x;
    const uint16_t* x1 = reinterpret_cast<const uint16_t*>(a.x) + row1 * a.ld_x;

    // ---- 1. my eighth of the width, 32 columns at a time, shared out among the warps ----
    const int k_slice = (a.width + kAdCluster * 32 - 1) / (kAdCluster * 32) * 32;
    const int k0 = static_cast<int>(cta) * k_slice, k1 = min(a.width, k0 + k_slice);
    const uint16_t* down = reinterpret_cast<const uint16_t*>(a.down) + static_cast<int64_t>(tile.x) * rank * a.width;
    for (int rb = 0; rb < rank; rb += NT * 8) {
        float acc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
#pragma unroll 2
        for (int k = k0 + kw * 32; k < k1; k += KW * 32) {
            const int kk = k + t * 8;
            const bool in = kk < k1;
            const uint4 xa = in && live0 ? *reinterpret_cast<const uint4*>(x0 + kk) : ad_zero();
            const uint4 xb = in && live1 ? *reinterpret_cast<const uint4*>(x1 + kk) : ad_zero();
            uint4 d[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j)
                d[j] = in && rb + j * 8 < rank ? ld_nc_v4(down + static_cast<int64_t>(rb + j * 8 + g) * a.width + kk) : ad_zero();
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                mma_m16n8k16<kBf16>(acc[j], xa.x, xb.x, xa.y, xb.y, d[j].x, d[j].y);
                mma_m16n8k16<kBf16>(acc[j], xa.z, xb.z, xa.w, xb.w, d[j].z, d[j].w);
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            *reinterpret_cast<float2*>(red + (warp * 16 + g) * 64 + j * 8 + 2 * t) = make_float2(acc[j][0], acc[j][1]);
            *reinterpret_cast<float2*>(red + (warp * 16 + g + 8) * 64 + j * 8 + 2 * t) = make_float2(acc[j][2], acc[j][3]);
        }
        __syncthreads();
        for (int i = tid; i < M * NT * 8; i += kAdThreads) {
            const int r = i / (NT * 8), c = i % (NT * 8);
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < KW; ++w) s += red[((w * MT + (r >> 4)) * 16 + (r & 15)) * 64 + c];
            part[r * 64 + c] = s;
        }
        // ---- 2. the eighths of the width meet: CTA r adds up eighth r of this block of h ----
        ad_cluster_sync();
        constexpr int QUADS = M * NT * 8 / 4;
        for (int i = tid; i < QUADS / kAdCluster; i += kAdThreads) {
            const int q = static_cast<int>(cta) * (QUADS / kAdCluster) + i;
            const int r = q / (NT * 2), c = q % (NT * 2) * 4;
            float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int p = 0; p < kAdCluster; ++p) {
                const float4 v = ad_load4(ad_at(part + r * 64 + c, p));
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
#pragma unroll
            for (int p = 0; p < kAdCluster; ++p) ad_store4(ad_at(h + r * padded + rb + c, p), s);
        }
        ad_cluster_sync();
    }
    // ---- h in two 16-bit parts ----
    if constexpr (!kBf16) {
        for (int r = warp; r < M; r += kAdWarps) {
            float m = 0.0f;
            for (int c = lane; c < rank; c += 32) m = fmaxf(m, fabsf(h[r * padded + c]));
            m = warp_max(m);
            int e = 0;
            if (m > 0.0f && m < INFINITY) frexpf(m, &e);
            if (lane == 0) row_scale[r] = ldexpf(1.0f, min(max(e - 9, -126), 126));
        }
        __syncthreads();
    }
    const int k_steps = (rank + 15) / 16;
    for (int i = tid; i < M * k_steps * 16; i += kAdThreads) {
        const int r = i / (k_steps * 16), c = i % (k_steps * 16);
        float v = c < rank ? h[r * padded + c] : 0.0f;
        if constexpr (!kBf16) v /= row_scale[r];
        const uint32_t hi = pack2<kBf16>(v, 0.0f);
        const float rest = v - unpack_lo<kBf16>(hi);
        h_hi[r * pitch + c] = static_cast<uint16_t>(hi);
        h_lo[r * pitch + c] = static_cast<uint16_t>(pack2<kBf16>(fabsf(rest) < INFINITY ? rest : 0.0f, 0.0f));
    }
    __syncthreads();
    // ---- 3. my eighth of the outputs, 32 columns at a time. Tile j, column 2 t + e of the MMA is column 8 t + 2 j + e of the 32 ----
    const uint16_t* up = reinterpret_cast<const uint16_t*>(a.up) + static_cast<int64_t>(tile.x) * a.outputs * rank;
    const float scale = a.scales[tile.x];
    float s0 = scale, s1 = scale;
    if constexpr (!kBf16) {
        s0 *= row_scale[r0];
        s1 *= row_scale[r1];
    }
    for (int n = n0 + kw * 32; n < n1; n += KW * 32) {
        const int col = n + t * 8;
        const bool in = col < n1;
        const uint16_t* b0 = reinterpret_cast<const uint16_t*>(a.base) + row0 * a.ld_base + col;
        const uint16_t* b1 = reinterpret_cast<const uint16_t*>(a.base) + row1 * a.ld_base + col;
        const uint4 base0 = in && live0 ? *reinterpret_cast<const uint4*>(b0) : ad_zero();
        const uint4 base1 = in && live1 ? *reinterpret_cast<const uint4*>(b1) : ad_zero();
        float acc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
        const int up_row = n + (g >> 1) * 8 + (g & 1);
        for (int ks = 0; ks < k_steps; ++ks) {
            const int c = ks * 16 + t * 4;
            uint2 u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                u[j] = up_row + 2 * j < n1 && c < rank ? *reinterpret_cast<const uint2*>(up + static_cast<int64_t>(up_row + 2 * j) * rank + c)
                                                       : make_uint2(0u, 0u);
            const uint2 p0 = *reinterpret_cast<const uint2*>(h_hi + r0 * pitch + c), p1 = *reinterpret_cast<const uint2*>(h_hi + r1 * pitch + c);
            const uint2 l0 = *reinterpret_cast<const uint2*>(h_lo + r0 * pitch + c), l1 = *reinterpret_cast<const uint2*>(h_lo + r1 * pitch + c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mma_m16n8k16<kBf16>(acc[j], p0.x, p1.x, p0.y, p1.y, u[j].x, u[j].y);
                mma_m16n8k16<kBf16>(acc[j], l0.x, l1.x, l0.y, l1.y, u[j].x, u[j].y);
            }
        }
        auto join = [&](const uint4& b, int e, float s) {
            return make_uint4(pack2<kBf16>(fmaf(s, acc[0][e], unpack_lo<kBf16>(b.x)), fmaf(s, acc[0][e + 1], unpack_hi<kBf16>(b.x))),
                              pack2<kBf16>(fmaf(s, acc[1][e], unpack_lo<kBf16>(b.y)), fmaf(s, acc[1][e + 1], unpack_hi<kBf16>(b.y))),
                              pack2<kBf16>(fmaf(s, acc[2][e], unpack_lo<kBf16>(b.z)), fmaf(s, acc[2][e + 1], unpack_hi<kBf16>(b.z))),
                              pack2<kBf16>(fmaf(s, acc[3][e], unpack_lo<kBf16>(b.w)), fmaf(s, acc[3][e + 1], unpack_hi<kBf16>(b.w))));
        };
        if (in && live0) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + row0 * a.ld_out + col) = join(base0, 0, s0);
        if (in && live1) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + row1 * a.ld_out + col) = join(base1, 2, s1);
    }
}

template <int MT, int NT, bool kBf16>
static int launch_adapters_as(const AdapterArgs& a, int n_tiles, cudaStream_t s) {
    auto kern = adapter_kernel<MT, NT, kBf16>;
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        HDS_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(ad_smem_bytes<MT>(kAdMaxRank))));
        configured[dev & 63] = true;
    }
    HDS_CHECK_CUDA(launch_kernel_cluster(kern, kAdCluster, dim3(static_cast<unsigned>(n_tiles) * kAdCluster), dim3(kAdThreads),
                                         ad_smem_bytes<MT>(a.rank), s, a));
    return HDS_OK;
}

template <int MT, bool kBf16>
static int launch_adapters(const AdapterArgs& a, int n_tiles, cudaStream_t s) {
    return a.rank <= 16 ? launch_adapters_as<MT, 2, kBf16>(a, n_tiles, s)
           : a.rank <= 32 ? launch_adapters_as<MT, 4, kBf16>(a, n_tiles, s) : launch_adapters_as<MT, 8, kBf16>(a, n_tiles, s);
}

}  // namespace hds

using namespace hds;

extern "C" int hds_adapter_add(const void* base, int64_t ld_base, const void* x, int64_t ld_x, const void* down, const void* up, const float* scales,
                               int n_adapters, int rank, int width, int outputs, const int32_t* order, const int32_t* tiles, int n_tiles,
                               int tile_rows, void* out, int64_t ld_out, int dtype, void* stream) {
    HDS_REQUIRE(dtype == 0 || dtype == 1, "adapter_add: dtype must be 0 (bf16) or 1 (fp16)");
    HDS_REQUIRE(rank >= 8 && rank <= kAdMaxRank && rank % 8 == 0, "adapter_add: ranks are multiples of 8 up to 256");
    HDS_REQUIRE(width > 0 && outputs > 0 && width % 8 == 0 && outputs % 8 == 0, "adapter_add: widths are multiples of 8");
    HDS_REQUIRE(ld_base % 8 == 0 && ld_x % 8 == 0 && ld_out % 8 == 0, "adapter_add: rows start on 16-byte boundaries");
    HDS_REQUIRE(((reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(down) |
                  reinterpret_cast<uintptr_t>(up) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(tiles)) & 15) == 0,
                "adapter_add: operands start on 16-byte boundaries");
    HDS_REQUIRE(tile_rows == 16 || tile_rows == 64, "adapter_add: tiles of 16 or 64 rows");
    HDS_REQUIRE(n_tiles >= 0 && n_tiles <= (1 << 26), "adapter_add: too many tiles");
    if (n_tiles == 0) return HDS_OK;
    AdapterArgs a;
    memset(&a, 0, sizeof(a));
    a.x = x; a.base = base; a.out = out; a.ld_x = ld_x; a.ld_base = ld_base; a.ld_out = ld_out;
    a.down = down; a.up = up; a.scales = scales; a.order = order; a.tiles = reinterpret_cast<const int4*>(tiles);
    a.n_adapters = n_adapters; a.rank = rank; a.width = width; a.outputs = outputs;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (tile_rows == 16) return dtype == 0 ? launch_adapters<1, true>(a, n_tiles, s) : launch_adapters<1, false>(a, n_tiles, s);
    return dtype == 0 ? launch_adapters<4, true>(a, n_tiles, s) : launch_adapters<4, false>(a, n_tiles, s);
}
