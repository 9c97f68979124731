// What a request lays on its logits before a token is chosen, in one pass over them:
//
//   x = x > 0 ? x / repetition : x * repetition       for tokens of its history (prompt and answer)
//   x -= frequency * count + presence * (count > 0)   count: how often the token stands in the answer
//   x += bias[token]                                  a list of tokens; of a token given twice the last one counts
//   x = -inf                                          where the grammar's mask has a zero bit
//
// A CTA takes a chunk of neighbouring logits of a row, asks for them, for their mask bits and for the history's first tokens, and writes the logits
// as they are, or as -inf, in their own type. It then counts the row's history into a table of the chunk in shared memory (per token: in the
// prompt, has a bias, count; integer atomics, so that the order does not matter); whoever finds a token untouched puts it on a list, and the
// listed tokens are computed and written, one per thread: a few hundred of a chunk of thousands, so that none of the streamed logits has to look
// into the table. In place works too: what a listed token is computed from is still there unless the mask hides it. Logits are read and
// written once; the history is read by every CTA of the row, from L2. A warp's ids that fall into the chunk, few of them, are queued up before they
// are counted, since a warp with one of them takes as long as one with 32; one lane asks for the list's places for a warp (a thousand
// threads at one counter took 4 us).
// A row may begin on any element: chunks are cut at 16-byte boundaries of the logits, so that all but a row's two ends are moved 16 bytes at a
// time.
//
// Measured (bytes that any form has to move, time, bytes per second; a copy runs at 6.55 TB/s):
//   1 row of 50272 (fp16), history of 700: 2.5 us, the chain of one CTA: ids, table, list
//   64 rows of 32000 (bf16), histories of up to 4096, 300 biases, masks: 9 MB, 13.0 us: a CTA counts 4096 ids for 8192 logits
//   256 rows of 131071 (fp32), histories of up to 8192, 64 biases, masks: 275 MB, 76.5 us, 3.6 TB/s: the same, in seven waves of CTAs, of whose 10 us
//   the logits are on the way for 3, and 73% of the issue slots; chunks of 16384 and 32768 take 74.9 and 70.0 us, but 17.6 and 28.1 at the 64 rows. Histories dealt out by chunk
//   in a kernel of its own beside the stream: 74.3 us, for two launches; CTAs that ask for their next chunk before they count this one's: 105 us, as
//   only two of them have registers
//
// No counterpart in the reference, which leaves the choice of tokens to its caller.
#include "hds_ptx.cuh"
#include "hds_host.cuh"
#include "../../../include/hds_b200.h"

namespace hds {

// Biases of a chunk kept in shared memory. The threads of a chunk with more search the row's whole list, which grows with its square: 64 rows of 32000
// take 8 us with 300 biases, 17 with 1000, 473 with 5000.
constexpr int kBiasPairs = 512;
constexpr int kQueue = 128;            // ids that a warp looks at in one go
constexpr int kNarrowCount = 0x3fff;   // what a count of 14 bits holds

struct ControlArgs {
    const void* x;
    void* out;
    int64_t ld_x, ld_out;
    int vocab, chunk, list;            // list: entries of the list of touched tokens
    const int32_t* history;            // [rows, ld_history]
    int64_t ld_history;
    int capacity;                      // history places of a row
    const int32_t* history_len;
    const int32_t* prompt_len;         // or nullptr: none of it is prompt
    const float* repetition;           // [rows] each, or nullptr
    const float* presence;
    const float* frequency;
    const int32_t* bias_ids;           // [rows, ld_bias_ids]; ids that are no token are passed over
    const float* bias;                 // [rows, ld_bias]
    int64_t ld_bias_ids, ld_bias;
    int n_bias;
    const uint32_t* mask;              // [n_masks, ld_mask] bits, a token's bit 1: allowed
    int64_t ld_mask;
    int n_masks;
    const int32_t* mask_rows;          // [rows] or nullptr (row i has mask i); a number that is no mask's: no grammar
};

template <int DT> struct ControlType { using type = uint16_t; };
template <> struct ControlType<2> { using type = uint32_t; };

// A token's entry of the table: 16 bits, or 32 for histories whose counts may need more than 14. Two entries of 16 bits share a word: counts
// stay below the flags, so that nothing is carried into the neighbour.
template <bool kWide>
struct ControlTable {
    static constexpr uint32_t kPrompt = kWide ? 0x80000000u : 0x8000u, kBias = kWide ? 0x40000000u : 0x4000u, kCount = kBias - 1u;
    uint32_t* words;
    // adds to the entry of place u (a count, or a flag) and returns what it was before
    __device__ __forceinline__ uint32_t touch(uint32_t u, bool count, uint32_t flag) const {
        if constexpr (kWide) return count ? atomicAdd(&words[u], 1u) : atomicOr(&words[u], flag);
        const uint32_t shift = (u & 1u) * 16u;
        return (count ? atomicAdd(&words[u >> 1], 1u << shift) : atomicOr(&words[u >> 1], flag << shift)) >> shift & 0xffffu;
    }
    __device__ __forceinline__ uint32_t at(uint32_t u) const {
        if constexpr (kWide) return words[u];
        return reinterpret_cast<const uint16_t*>(words)[u];
    }
};
// the table, the biases of the chunk (place, number in the row's list), the warps' queues, the list of touched tokens
__host__ __device__ constexpr int control_table_bytes(int chunk, bool wide) { return chunk * (wide ? 4 : 2); }
inline int control_smem_bytes(const ControlArgs& a, bool wide, int threads) {
    return control_table_bytes(a.chunk, wide) + kBiasPairs * 8 + threads / 32 * kQueue * 4 + (a.list * 2 + 15) / 16 * 16;
}

template <int DT>
__device__ __forceinline__ void control_store(void* base, int64_t i, float v) {
    if constexpr (DT == 2) reinterpret_cast<float*>(base)[i] = v;
    else store_scalar<DT == 0>(base, i, v);
}

// THREADS threads with PER logits each
template <int DT, int THREADS, int PER, bool kWide>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 4 : 12) logit_controls_kernel(const ControlArgs a) {
    using T = typename ControlType<DT>::type;
    using Table = ControlTable<kWide>;
    constexpr int E = 16 / static_cast<int>(sizeof(T));   // logits per 16 bytes
    constexpr int VECS = PER / E;
    constexpr uint32_t CHUNK = THREADS * PER;
    constexpr T kHidden = static_cast<T>(DT == 0 ? 0xff80u : DT == 1 ? 0xfc00u : 0xff800000u);     // -inf
    extern __shared__ __align__(16) uint8_t control_smem[];
    __shared__ int n_listed, n_pairs;
    pdl_enter();
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld_x;
    T* out = reinterpret_cast<T*>(a.out) + row * a.ld_out;
    // tokens are counted from the 16-byte boundary at or before the row's first logit
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const bool wide_out = (reinterpret_cast<uintptr_t>(out) & 15) == (reinterpret_cast<uintptr_t>(x) & 15);
    const int first = static_cast<int>(blockIdx.x * CHUNK) - off;        // the chunk's first token; may be below 0
    if (first >= a.vocab) return;
    // whole vectors of the chunk: from `lead` on, up to `whole`
    const int lead = first < 0 ? 1 : 0, whole = min(static_cast<int>(CHUNK) / E, (a.vocab - first) / E);

    uint4 raw[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int q = tid + i * THREADS;
        if (q >= lead && q < whole) raw[i] = *reinterpret_cast<const uint4*>(x + first + q * E);
    }
    const uint32_t* mask = nullptr;
    if (a.mask) {
        const int m = a.mask_rows ? a.mask_rows[row] : row;
        if (m >= 0 && m < a.n_masks) mask = a.mask + m * a.ld_mask;
    }
    uint32_t bits[VECS];
    if (mask) {
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            const int q = tid + i * THREADS, v = first + q * E;
            if (q >= lead && q < whole) bits[i] = __funnelshift_r(mask[v >> 5], mask[(v + E - 1) >> 5], v & 31);
        }
    }
    const float rep = a.repetition ? a.repetition[row] : 1.0f;
    const float pres = a.presence ? a.presence[row] : 0.0f, freq = a.frequency ? a.frequency[row] : 0.0f;
    int told = a.history ? min(max(a.history_len[row], 0), a.capacity) : 0;
    if (rep == 1.0f && pres == 0.0f && freq == 0.0f) told = 0;
    const bool any = told > 0 || a.n_bias > 0;
    const Table table{reinterpret_cast<uint32_t*>(control_smem)};
    int2* pairs = reinterpret_cast<int2*>(control_smem + control_table_bytes(CHUNK, kWide));
    uint32_t* queue = reinterpret_cast<uint32_t*>(pairs + kBiasPairs) + (tid >> 5) * kQueue;
    uint16_t* listed = reinterpret_cast<uint16_t*>(reinterpret_cast<uint32_t*>(pairs + kBiasPairs) + THREADS / 32 * kQueue);
    auto allowed = [&](int v) { return mask == nullptr || (mask[v >> 5] >> (v & 31) & 1u); };
    // a warp's next ids, four per lane
    const int32_t* h = a.history + row * a.ld_history;
    const bool wide = (reinterpret_cast<uintptr_t>(h) & 15) == 0;
    auto ask = [&](int j) {
        if (wide && j + 4 <= told) return *reinterpret_cast<const int4*>(h + j);
        return make_int4(j < told ? h[j] : first - 1, j + 1 < told ? h[j + 1] : first - 1, j + 2 < told ? h[j + 2] : first - 1, j + 3 < told ? h[j + 3] : first - 1);
    };
    int j0 = (tid >> 5) * kQueue;
    int4 next = make_int4(0, 0, 0, 0);
    if (any) {
        if (told > 0) next = ask(j0 + 4 * lane);
        for (int i = tid; i < control_table_bytes(CHUNK, kWide) / 16; i += THREADS) reinterpret_cast<uint4*>(control_smem)[i] = make_uint4(0u, 0u, 0u, 0u);
        if (tid == 0) n_listed = n_pairs = 0;
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int q = tid + i * THREADS;
        if (q < lead || q >= whole) continue;
        const int v = first + q * E;
        uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        if (mask) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (DT == 2) {
                    if (!(bits[i] >> e & 1u)) w[e] = kHidden;
                } else {
                    if (!(bits[i] >> (2 * e) & 1u)) w[e] = (w[e] & 0xffff0000u) | kHidden;
                    if (!(bits[i] >> (2 * e + 1) & 1u)) w[e] = (w[e] & 0xffffu) | static_cast<uint32_t>(kHidden) << 16;
                }
            }
        }
        if (wide_out) {
            *reinterpret_cast<uint4*>(out + v) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) out[v + e] = static_cast<T>(DT == 2 ? w[e % 4] : w[e / 2] >> 16 * (e & 1));
        }
    }
    // a row's two ends inside vectors
    if (lead && tid < E - off && tid < a.vocab) out[tid] = allowed(tid) ? x[tid] : kHidden;
    if (whole * E < static_cast<int>(CHUNK) && (whole > 0 || !lead)) {
        const int v = first + whole * E + tid;
        if (tid < E && v >= 0 && v < a.vocab) out[v] = allowed(v) ? x[v] : kHidden;
    }
    if (any) {
        __syncthreads();
        // (ids that are no tokens fall outside the chunk, or on places of it that nobody reads: below 0 and from the vocabulary's end on)
        // (a warp together: one of its lanes asks for the list's places)
        auto touch = [&](bool in, uint32_t u, bool count, uint32_t flag) {
            const bool fresh = in && table.touch(u, count, flag) == 0u;
            const uint32_t who = __ballot_sync(0xffffffffu, fresh);
            int at = 0;
            if (lane == 0 && who) at = atomicAdd(&n_listed, __popc(who));
            at = __shfl_sync(0xffffffffu, at, 0);
            if (fresh) listed[at + __popc(who & ((1u << lane) - 1u))] = static_cast<uint16_t>(u);
        };
        if (told > 0) {
            const int prompt = a.prompt_len ? a.prompt_len[row] : 0;
            for (; j0 < told; j0 += THREADS * 4) {      // (a warp together)
                const int j = j0 + 4 * lane;
                const int32_t id[4] = {next.x, next.y, next.z, next.w};
                next = ask(j + THREADS * 4);
                int n = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t u = static_cast<uint32_t>(id[k]) - static_cast<uint32_t>(first);
                    const bool in = u < CHUNK;
                    const uint32_t who = __ballot_sync(0xffffffffu, in);
                    if (in) queue[n + __popc(who & ((1u << lane) - 1u))] = j + k < prompt ? u | 0x80000000u : u;
                    n += __popc(who);
                }
                __syncwarp();
                for (int k0 = 0; k0 < n; k0 += 32) {
                    const uint32_t w = k0 + lane < n ? queue[k0 + lane] : 0u;
                    touch(k0 + lane < n, w & 0x7fffffffu, !(w >> 31), Table::kPrompt);
                }
                __syncwarp();
            }
        }
        const int32_t* ids = a.bias_ids + row * a.ld_bias_ids;
        for (int b0 = tid - lane; b0 < a.n_bias; b0 += THREADS) {
            const int b = b0 + lane;
            const uint32_t u = static_cast<uint32_t>(b < a.n_bias ? ids[b] : first - 1) - static_cast<uint32_t>(first);
            touch(u < CHUNK, u, false, Table::kBias);
            if (u < CHUNK) {
                const int at = atomicAdd(&n_pairs, 1);
                if (at < kBiasPairs) pairs[at] = make_int2(static_cast<int>(u), b);
            }
        }
    }
    if (!any) return;
    __syncthreads();
    const int n = n_listed, np = n_pairs;
    for (int i = tid; i < n; i += THREADS) {
        const int u = listed[i], v = first + u;
        if (v < 0 || v >= a.vocab || !allowed(v)) continue;
        const uint32_t w = table.at(u);
        float f = load_any<DT>(x, v);
        if (w & ~Table::kBias) {
            f = f > 0.0f ? f / rep : f * rep;
            const uint32_t c = w & Table::kCount;
            if (c) f = f - freq * static_cast<float>(c) - pres;
        }
        if (w & Table::kBias) {      // the last one of this token
            int last = -1;
            if (np <= kBiasPairs) {
                for (int k = 0; k < np; ++k) last = pairs[k].x == u ? max(last, pairs[k].y) : last;
            } else {
                const int32_t* ids = a.bias_ids + row * a.ld_bias_ids;
                for (int k = 0; k < a.n_bias; ++k) last = ids[k] == v ? k : last;
            }
            f += a.bias[row * a.ld_bias + last];
        }
        control_store<DT>(out, v, f);
    }
}

template <int DT, int THREADS, int PER, bool kWide>
static int launch_controls_as(ControlArgs a, int rows, cudaStream_t s) {
    auto kern = logit_controls_kernel<DT, THREADS, PER, kWide>;
    a.chunk = THREADS * PER;
    a.list = static_cast<int>(a.chunk < static_cast<int64_t>(a.capacity) + a.n_bias ? a.chunk : static_cast<int64_t>(a.capacity) + a.n_bias);
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        ControlArgs most = a;
        most.list = a.chunk;
        HDS_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, control_smem_bytes(most, kWide, THREADS)));
        configured[dev & 63] = true;
    }
    const int extra = 16 / (DT == 2 ? 4 : 2) - 1;       // places ahead of the first logit, at most
    const int chunks = (a.vocab + extra + a.chunk - 1) / a.chunk;
    const size_t smem = a.history != nullptr || a.n_bias > 0 ? control_smem_bytes(a, kWide, THREADS) : 0;
    HDS_CHECK_CUDA(launch_kernel(kern, dim3(chunks, rows), dim3(THREADS), smem, s, a));
    return HDS_OK;
}

template <int DT, bool kWide>
static int launch_controls(const ControlArgs& a, int rows, cudaStream_t s) {
    // Every CTA of a row looks at all of its history: chunks of 8192 where there is more of it than a small chunk is worth, and SMs are filled.
    // Measured: 256 rows of 131071 fp32 logits, histories of up to 8192 and 64 biases 76 us with chunks of 8192 and 121 with 2048, 64 of 32000 in
    // bf16, 4096 and 300 12.7 and 17.0; 103 of 10202 in fp32 and 317 5.6 and 4.9, 1 of 50272 and 700 2.7 and 2.5.
    if (static_cast<int64_t>(rows) * ((a.vocab + 8191) / 8192) >= sm_count() && a.capacity + a.n_bias >= 1024)
        return launch_controls_as<DT, 512, 16, kWide>(a, rows, s);
    return launch_controls_as<DT, 128, 16, kWide>(a, rows, s);
}

}  // namespace hds

using namespace hds;

extern "C" int hds_logit_controls(const void* logits, int64_t ld_logits, void* out, int64_t ld_out, int rows, int vocab, const int32_t* history,
                                  int64_t ld_history, int capacity, const int32_t* history_len, const int32_t* prompt_len, const float* repetition,
                                  const float* presence, const float* frequency, const int32_t* bias_ids, int64_t ld_bias_ids, const float* bias,
                                  int64_t ld_bias, int n_bias, const uint32_t* mask, int64_t ld_mask, int n_masks, const int32_t* mask_rows,
                                  int dtype, void* stream) {
    HDS_REQUIRE(dtype >= 0 && dtype <= 2, "logit_controls: dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    HDS_REQUIRE(rows >= 0 && rows <= 65535 && vocab >= 0 && vocab < (1 << 30), "logit_controls: rows in [0, 65535] and a vocabulary below 2^30");
    HDS_REQUIRE(n_bias >= 0 && capacity >= 0 && capacity < (1 << 30) && n_masks >= 0, "logit_controls: sizes in [0, 2^30)");
    HDS_REQUIRE(history == nullptr || history_len != nullptr, "logit_controls: a history needs its lengths");
    HDS_REQUIRE(mask == nullptr || ld_mask >= (static_cast<int64_t>(vocab) + 31) / 32, "logit_controls: a mask has a bit per token");
    HDS_REQUIRE(rows <= 1 || ld_out >= vocab, "logit_controls: rows of out share memory");
    const int elem = dtype == 2 ? 4 : 2;
    HDS_REQUIRE(reinterpret_cast<uintptr_t>(logits) % elem == 0 && reinterpret_cast<uintptr_t>(out) % elem == 0, "logit_controls: logits on odd addresses");
    if (rows == 0 || vocab == 0) return HDS_OK;
    ControlArgs a;
    memset(&a, 0, sizeof(a));
    a.x = logits; a.out = out; a.ld_x = ld_logits; a.ld_out = ld_out; a.vocab = vocab;
    a.history = history; a.ld_history = ld_history; a.capacity = capacity; a.history_len = history_len; a.prompt_len = prompt_len;
    a.repetition = repetition; a.presence = presence; a.frequency = frequency;
    a.bias_ids = bias_ids; a.ld_bias_ids = ld_bias_ids; a.bias = bias; a.ld_bias = ld_bias;
    a.n_bias = bias_ids != nullptr && bias != nullptr ? n_bias : 0;
    a.mask = mask; a.ld_mask = ld_mask; a.n_masks = n_masks; a.mask_rows = mask_rows;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (capacity > kNarrowCount)
        return dtype == 0 ? launch_controls<0, true>(a, rows, s) : dtype == 1 ? launch_controls<1, true>(a, rows, s) : launch_controls<2, true>(a, rows, s);
    return dtype == 0 ? launch_controls<0, false>(a, rows, s) : dtype == 1 ? launch_controls<1, false>(a, rows, s) : launch_controls<2, false>(a, rows, s);
}
