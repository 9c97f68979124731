// What a request lays on its logits before a token is chosen, in one pass over them:
//
//   x = x > 0 ? x / repetition : x * repetition       for tokens of its history (prompt and answer)
//   x -= frequency * count + presence * (count > 0)   count: how often the token stands in the answer
//   x += bias[token]                                  a list of tokens; of a token given twice the last one counts
//   x = -inf                                          where the grammar's mask has a zero bit
//
// A CTA takes `chunk` neighbouring logits of a row. It asks for them first (they wait in registers), counts the row's history into a table of
// the chunk in shared memory meanwhile (one word per token: bit 31 in the prompt, the rest counts; integer atomics, so that the order
// does not matter), and then writes what comes out. Logits are read and written once; the history is read by every CTA of the row, from L2.
// A row may begin on any element: chunks are cut at 16-byte boundaries of the logits, so that all but a row's two ends are moved 16 bytes at a
// time. Value e of vector i has its word at e * (chunk / E) + i, where neighbouring lanes meet no bank twice.
//
// No counterpart in the reference, which leaves the choice of tokens to its caller.
#include "hds_ptx.cuh"
#include "hds_host.cuh"
#include "../../../include/hds_b200.h"

namespace hds {

constexpr int kControlPer = 16;        // logits per thread
constexpr uint32_t kInPrompt = 0x80000000u;

struct ControlArgs {
    const void* x;
    void* out;
    int64_t ld_x, ld_out;
    int vocab, chunk;
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

template <int DT>
__device__ __forceinline__ void control_unpack(const uint4& v, float (&f)[DT == 2 ? 4 : 8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == 2) {
            f[i] = __uint_as_float(w[i]);
        } else {
            f[2 * i] = unpack_lo<DT == 0>(w[i]);
            f[2 * i + 1] = unpack_hi<DT == 0>(w[i]);
        }
    }
}
template <int DT>
__device__ __forceinline__ uint4 control_pack(const float (&f)[DT == 2 ? 4 : 8]) {
    if constexpr (DT == 2) return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    else return make_uint4(pack2<DT == 0>(f[0], f[1]), pack2<DT == 0>(f[2], f[3]), pack2<DT == 0>(f[4], f[5]), pack2<DT == 0>(f[6], f[7]));
}
template <int DT>
__device__ __forceinline__ void control_store(void* base, int64_t i, float v) {
    if constexpr (DT == 2) reinterpret_cast<float*>(base)[i] = v;
    else store_scalar<DT == 0>(base, i, v);
}

template <int DT>
__global__ void __launch_bounds__(512) logit_controls_kernel(const ControlArgs a) {
    using T = typename ControlType<DT>::type;
    constexpr int E = 16 / static_cast<int>(sizeof(T));   // logits per 16 bytes
    constexpr int VECS = kControlPer / E;
    extern __shared__ uint32_t control_smem[];
    pdl_enter();
    const int row = blockIdx.y, tid = threadIdx.x, threads = blockDim.x, vecs = a.chunk / E;
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld_x;
    T* out = reinterpret_cast<T*>(a.out) + row * a.ld_out;
    // places are counted from the 16-byte boundary at or before the row's first logit, which has place `off`
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const bool wide_out = (reinterpret_cast<uintptr_t>(out) & 15) == (reinterpret_cast<uintptr_t>(x) & 15);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * a.chunk - off;      // token of the chunk's place 0; may be below 0
    if (first >= a.vocab) return;

    uint4 raw[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int64_t v = first + static_cast<int64_t>(tid + i * threads) * E;
        if (v >= 0 && v + E <= a.vocab) raw[i] = *reinterpret_cast<const uint4*>(x + v);
    }
    const float rep = a.repetition ? a.repetition[row] : 1.0f;
    const float pres = a.presence ? a.presence[row] : 0.0f, freq = a.frequency ? a.frequency[row] : 0.0f;
    const int told = a.history ? min(max(a.history_len[row], 0), a.capacity) : 0;
    const bool counts = told > 0 && !(rep == 1.0f && pres == 0.0f && freq == 0.0f);
    const uint32_t* mask = nullptr;
    if (a.mask) {
        const int m = a.mask_rows ? a.mask_rows[row] : row;
        if (m >= 0 && m < a.n_masks) mask = a.mask + m * a.ld_mask;
    }
    uint32_t* seen = control_smem;                                                           // [chunk]
    int32_t* given = reinterpret_cast<int32_t*>(control_smem + (a.history ? a.chunk : 0));  // [chunk]: 1 + place in the list of biases
    for (int i = tid; i < a.chunk; i += threads) {
        if (counts) seen[i] = 0u;
        if (a.n_bias) given[i] = 0;
    }
    __syncthreads();
    auto place = [&](int32_t id) {       // of a token's word, or -1 outside this chunk
        const int64_t u = id - first;
        if (id < 0 || id >= a.vocab || u < 0 || u >= a.chunk) return -1;
        return static_cast<int>(u) % E * vecs + static_cast<int>(u) / E;
    };
    if (counts) {
        const int32_t* h = a.history + row * a.ld_history;
        const int prompt = a.prompt_len ? a.prompt_len[row] : 0;
        for (int j = tid; j < told; j += 4 * threads) {
            int32_t id[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) id[k] = j + k * threads < told ? h[j + k * threads] : -1;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int p = place(id[k]);
                if (p < 0) continue;
                if (j + k * threads < prompt) atomicOr(&seen[p], kInPrompt);
                else atomicAdd(&seen[p], 1u);
            }
        }
    }
    for (int j = tid; j < a.n_bias; j += threads) {
        const int p = place(a.bias_ids[row * a.ld_bias_ids + j]);
        if (p >= 0) atomicMax(&given[p], j + 1);
    }
    __syncthreads();
    auto apply = [&](float f, int p) {
        if (counts) {
            const uint32_t w = seen[p];
            if (w) {
                f = f > 0.0f ? f / rep : f * rep;
                const uint32_t c = w & ~kInPrompt;
                if (c) f = f - freq * static_cast<float>(c) - pres;
            }
        }
        if (a.n_bias) {
            const int j = given[p];
            if (j) f += a.bias[row * a.ld_bias + j - 1];
        }
        return f;
    };
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int q = tid + i * threads;                       // vector of the chunk
        const int64_t v = first + static_cast<int64_t>(q) * E;
        if (v >= 0 && v + E <= a.vocab) {
            float f[E];
            control_unpack<DT>(raw[i], f);
            if (counts || a.n_bias) {
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] = apply(f[e], e * vecs + q);
            }
            if (mask) {
                const int w = static_cast<int>(v >> 5), s = static_cast<int>(v & 31);
                uint32_t bits = mask[w] >> s;
                if (s + E > 32) bits |= mask[w + 1] << (32 - s);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (!(bits >> e & 1u)) f[e] = -INFINITY;
            }
            if (wide_out) {
                *reinterpret_cast<uint4*>(out + v) = control_pack<DT>(f);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) control_store<DT>(out, v + e, f[e]);
            }
        } else {      // a row's end inside a vector
            for (int e = 0; e < E; ++e) {
                if (v + e < 0 || v + e >= a.vocab) continue;
                float f = apply(load_any<DT>(x, v + e), e * vecs + q);
                if (mask && !(mask[(v + e) >> 5] >> ((v + e) & 31) & 1u)) f = -INFINITY;
                control_store<DT>(out, v + e, f);
            }
        }
    }
}

template <int DT>
static int launch_controls(const ControlArgs& a, int rows, cudaStream_t s) {
    const int64_t smem = static_cast<int64_t>(a.chunk) * 4 * ((a.history != nullptr) + (a.n_bias > 0));
    auto kern = logit_controls_kernel<DT>;
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        HDS_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 65536));
        configured[dev & 63] = true;
    }
    const int extra = 16 / (DT == 2 ? 4 : 2) - 1;       // places ahead of the first logit, at most
    const int64_t chunks = (static_cast<int64_t>(a.vocab) + extra + a.chunk - 1) / a.chunk;
    HDS_CHECK_CUDA(launch_kernel(kern, dim3(static_cast<unsigned>(chunks), rows), dim3(a.chunk / kControlPer), static_cast<size_t>(smem), s, a));
    return HDS_OK;
}

}  // namespace hds

using namespace hds;

extern "C" int hds_logit_controls(const void* logits, int64_t ld_logits, void* out, int64_t ld_out, int rows, int vocab, const int32_t* history,
                                  int64_t ld_history, int capacity, const int32_t* history_len, const int32_t* prompt_len, const float* repetition,
                                  const float* presence, const float* frequency, const int32_t* bias_ids, int64_t ld_bias_ids, const float* bias,
                                  int64_t ld_bias, int n_bias, const uint32_t* mask, int64_t ld_mask, int n_masks, const int32_t* mask_rows,
                                  int dtype, void* stream) {
    HDS_REQUIRE(dtype >= 0 && dtype <= 2, "logit_controls: dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    HDS_REQUIRE(rows >= 0 && rows <= 65535 && vocab >= 0, "logit_controls: rows in [0, 65535] and a vocabulary of at least 0");
    HDS_REQUIRE(n_bias >= 0 && capacity >= 0 && n_masks >= 0, "logit_controls: negative size");
    HDS_REQUIRE(history == nullptr || history_len != nullptr, "logit_controls: a history needs its lengths");
    HDS_REQUIRE(mask == nullptr || ld_mask >= (static_cast<int64_t>(vocab) + 31) / 32, "logit_controls: a mask has a bit per token");
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
    a.chunk = static_cast<int64_t>(rows) * ((vocab + 8191) / 8192) >= sm_count() ? 8192 : 2048;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == 0 ? launch_controls<0>(a, rows, s) : dtype == 1 ? launch_controls<1>(a, rows, s) : launch_controls<2>(a, rows, s);
}
