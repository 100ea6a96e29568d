// What stands between a model's logits and the probabilities that words are drawn from or drafts verified against: penalties for repeated words, biases, temperature,
// a grammar's mask.  Of a row with history h (the first of it a prompt), word w, n(w) its times behind the prompt:
//
//   z = z / repetition (z > 0) or z * repetition, where w is in h;   z -= frequency * n(w) + presence, where n(w) > 0
//   z += its biases, one after the other;   z *= 1 / temperature;   -inf, where the mask has no bit for w
//
// A cluster of CTAs has the row, a CTA a piece of the vocabulary with a 32-bit word for each: how often, whether in the history, whether there is a bias.  The CTAs read a share
// of the history each and count into the piece's owner by atomics over the cluster's shared memory: the history is read once, whatever the vocabulary's size is, and whole numbers add
// up the same in every order.  Equal words of a warp's 32 are counted by one lane, so that a history of one word only does not queue up.  The logits' first loads are on
// their way meanwhile.  Biases of a piece stand in a list in their order, which is only gone through for words that are marked.
#include "paged.cuh"
#include "tc2_common.cuh"

namespace zl {

constexpr int kAlMaxCluster = 8, kAlList = 512, kAlMaxPiece = 49152;
constexpr uint32_t kAlSeen = 0x80000000u, kAlBias = 0x40000000u, kAlCount = 0x3fffffffu;

struct AdjustLogits {
    const void* in;
    void* out;
    long long ld_in, ld_out;
    const int32_t *tokens, *token_seq, *token_lens, *prompt_lens, *bias_starts, *bias_words, *mask, *mask_row;
    const float *repetition, *frequency, *presence, *bias, *temperature;
    long long ld_tokens, ld_mask;
    int seqs, longest, n_bias, masks, vocab, ctas, parts, piece;
    PagedDivisor by_piece;
};

template <typename TI, int VEC>
__device__ __forceinline__ void al_load(TI (&v)[VEC], const TI* at) {
    if constexpr (VEC * sizeof(TI) == 16) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(at);
    else
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = at[i];
}

// dynamic shared memory: a word for each of the piece's, where there is a history or a bias
template <typename TI, typename TO, int VEC>
__global__ void __launch_bounds__(512) k_adjust_logits(const AdjustLogits p) {
    constexpr int kAhead = VEC == 1 ? 8 : 2;
    extern __shared__ __align__(16) uint32_t al_count[];
    __shared__ int s_words[kAlList], s_listed;
    __shared__ float s_bias[kAlList];
    const int tid = threadIdx.x, lane = tid & 31, threads = blockDim.x;
    const int rank = blockIdx.x % p.ctas, part = blockIdx.x / p.ctas % p.parts, r = blockIdx.x / (p.ctas * p.parts);
    const int lo0 = part * p.ctas * p.piece, lo = min(lo0 + rank * p.piece, p.vocab), hi = min(lo + p.piece, p.vocab);   // the cluster's first word; this CTA's
    const bool counts = p.tokens != nullptr, marks = counts || p.bias_starts;
    if (marks) {
        for (int i = tid * 4; i < hi - lo; i += threads * 4) *reinterpret_cast<uint4*>(al_count + i) = make_uint4(0, 0, 0, 0);
        if (counts && p.ctas > 1) cluster_arrive();
        else __syncthreads();
    }
    pdl_trigger();
    pdl_wait();
    const TI* in = static_cast<const TI*>(p.in) + (long long)r * p.ld_in;
    TO* out = static_cast<TO*>(p.out) + (long long)r * p.ld_out;
    TI x[kAhead][VEC];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * threads * VEC;
            if (i < hi) al_load(x[u], in + i);
        }
    };
    fetch(lo + tid * VEC);
    const float rep = p.repetition ? p.repetition[r] : 1.f, freq = p.frequency ? p.frequency[r] : 0.f, pres = p.presence ? p.presence[r] : 0.f;
    const float heat = p.temperature ? p.temperature[r] : 0.f, inv = heat >= 1.17549435e-38f ? 1.f / heat : 1.f;
    const int mask_row = !p.mask ? -1 : p.mask_row ? p.mask_row[r] : r;
    const int32_t* mask = mask_row >= 0 && mask_row < p.masks ? p.mask + (long long)mask_row * p.ld_mask : nullptr;
    int first = 0, last = 0;   // of the biases
    if (p.bias_starts) first = max(p.bias_starts[r], 0), last = min(p.bias_starts[r + 1], p.n_bias);
    if (counts) {
        const int seq = p.token_seq ? p.token_seq[r] : r, n = seq >= 0 && seq < p.seqs ? min(p.token_lens[r], p.longest) : 0, prompt = p.prompt_lens ? p.prompt_lens[r] : 0;
        const int32_t* words = p.tokens + (long long)max(seq, 0) * p.ld_tokens;
        if (p.ctas > 1) cluster_wait();
        for (int i0 = rank * threads + (tid & ~31); i0 < n; i0 += p.ctas * threads) {
            const int i = i0 + lane, word = i < n ? words[i] : -1, off = word - lo0, owner = word >= lo0 && word < p.vocab ? p.by_piece(off) : p.ctas;
            const bool is = owner < p.ctas, behind = i >= prompt;
            const unsigned same = __match_any_sync(0xffffffffu, is ? off << 1 | (int)behind : -1);
            if (is && (same & ((1u << lane) - 1u)) == 0) {
                uint32_t at = smem_u32(al_count + (off - owner * p.piece));
                if (p.ctas > 1) at = cluster_map(at, (uint32_t)owner);
                if (behind) asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(at), "r"((uint32_t)__popc(same)) : "memory");
                else asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(at), "r"(kAlSeen) : "memory");
            }
        }
    }
    if (tid < 32 && p.bias_starts) {
        int listed = 0;
        for (int i0 = first; i0 < last; i0 += 32) {
            const int i = i0 + lane, word = i < last ? p.bias_words[i] : -1;
            const bool is = word >= lo && word < hi;
            const unsigned here = __ballot_sync(0xffffffffu, is);
            const int at = listed + __popc(here & ((1u << lane) - 1u));
            if (is) {
                atomicOr(al_count + (word - lo), kAlBias);
                if (at < kAlList) s_words[at] = word, s_bias[at] = p.bias[i];
            }
            listed += __popc(here);
        }
        if (lane == 0) s_listed = listed;
    }
    if (counts && p.ctas > 1) cluster_sync_all();
    else if (marks) __syncthreads();
    for (int i0 = lo + tid * VEC; i0 < hi; i0 += kAhead * threads * VEC) {
        if (i0 != lo + tid * VEC) fetch(i0);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * threads * VEC;
            if (i >= hi) break;
            const uint32_t allowed = mask ? (uint32_t)mask[i >> 5] >> (i & 31) : 0xffffffffu;
            uint32_t mark[VEC] = {};
            if (marks) {
                if constexpr (VEC % 4 == 0)
#pragma unroll
                    for (int e = 0; e < VEC; e += 4) *reinterpret_cast<uint4*>(mark + e) = *reinterpret_cast<const uint4*>(al_count + (i - lo) + e);
                else
                    mark[0] = al_count[i - lo];
            }
            TO y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float z = to_f32<TI>(x[u][e]);
                if (mark[e]) {
                    const uint32_t n = mark[e] & kAlCount;
                    if (n || (mark[e] & kAlSeen)) z = z > 0.f ? z / rep : z * rep;
                    if (n) z = z - freq * (float)n - pres;
                    if (mark[e] & kAlBias) {
                        if (s_listed <= kAlList) {
                            for (int b = 0; b < s_listed; ++b)
                                if (s_words[b] == i + e) z += s_bias[b];
                        } else {
                            for (int b = first; b < last; ++b)
                                if (p.bias_words[b] == i + e) z += p.bias[b];
                        }
                    }
                }
                y[e] = from_f32<TO>(allowed >> e & 1u ? z * inv : -INFINITY);
            }
            if constexpr (VEC == 1) out[i] = y[0];
            else
#pragma unroll
                for (int e = 0; e < VEC * (int)sizeof(TO); e += 16) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out + i) + e) = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(y) + e);
        }
    }
}

template <typename TI, typename TO>
static int adjust_logits(const AdjustLogits& p, int rows, bool pdl, zl_stream_t stream) {
    // whole 16 bytes where rows and pitches allow it
    constexpr int kVec = 16 / sizeof(TI);
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.in) | reinterpret_cast<uintptr_t>(p.out);
    const bool wide = at % 16 == 0 && p.vocab % kVec == 0 && p.ld_in * sizeof(TI) % 16 == 0 && p.ld_out * sizeof(TO) % 16 == 0;
    auto kernel = wide ? k_adjust_logits<TI, TO, kVec> : k_adjust_logits<TI, TO, 1>;
    const size_t smem = p.tokens || p.bias_starts ? (size_t)p.piece * 4 : 0;
    static bool done[2][64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !done[wide][dev]) {
        ZL_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kAlMaxPiece * 4));
        if (dev >= 0 && dev < 64) done[wide][dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.ctas * p.parts) * rows);
    cfg.blockDim = dim3(p.piece > 8192 ? 512 : 256);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (p.ctas > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = p.ctas;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    zl_count_launch();
    ZL_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return ZL_OK;
}

}  // namespace zl

using namespace zl;

extern "C" int zl_adjust_logits(const void* logits, long long ld_logits, int dtype, void* out, long long ld_out, int out_dtype, int rows, int vocab,
                                const int32_t* tokens, long long ld_tokens, int seqs, int longest, const int32_t* token_seq, const int32_t* token_lens,
                                const int32_t* prompt_lens, const float* repetition, const float* frequency, const float* presence, const int32_t* bias_starts,
                                const int32_t* bias_words, const float* bias, int n_bias, const float* temperature, const int32_t* mask, long long ld_mask,
                                int masks, const int32_t* mask_row, int pdl, zl_stream_t stream) {
    ZL_CHECK_ARG(logits && out && rows > 0 && vocab > 0 && ld_logits >= vocab && ld_out >= vocab);
    ZL_CHECK_ARG(!tokens || (token_lens && seqs > 0 && longest >= 0 && ld_tokens >= longest && (token_seq || seqs >= rows)));
    ZL_CHECK_ARG(!bias_starts || (n_bias >= 0 && (n_bias == 0 || (bias_words && bias))));
    ZL_CHECK_ARG(!mask || (masks > 0 && ld_mask >= (vocab - 1) / 32 + 1 && (mask_row || masks >= rows)));
    ZL_CHECK_SUPPORTED(vocab <= 1 << 24 && longest <= 1 << 29 && (out_dtype == dtype || out_dtype == ZL_F32));
    AdjustLogits p = {logits, out, ld_logits, ld_out, tokens, token_seq, token_lens, prompt_lens, bias_starts, bias_words, mask, mask_row,
                      repetition, frequency, presence, bias, temperature, ld_tokens, ld_mask, seqs, longest, n_bias, masks, vocab};
    // Eight CTAs of 2048 words or more
    p.ctas = 1;
    while (p.ctas < kAlMaxCluster && p.ctas * 2048 < vocab) p.ctas *= 2;
    p.parts = (vocab - 1) / (p.ctas * kAlMaxPiece) + 1;
    p.piece = (int)((((long long)vocab - 1) / (p.ctas * p.parts) + 32) / 32 * 32);
    p.by_piece = paged_divisor(p.piece);
    ZL_CHECK_SUPPORTED((long long)rows * p.ctas * p.parts < 1ll << 31);
    if (dtype == ZL_F32) return adjust_logits<float, float>(p, rows, pdl != 0, stream);
    if (dtype == ZL_F16) return out_dtype == ZL_F32 ? adjust_logits<__half, float>(p, rows, pdl != 0, stream) : adjust_logits<__half, __half>(p, rows, pdl != 0, stream);
    ZL_CHECK_SUPPORTED(dtype == ZL_BF16);
    return out_dtype == ZL_F32 ? adjust_logits<__nv_bfloat16, float>(p, rows, pdl != 0, stream) : adjust_logits<__nv_bfloat16, __nv_bfloat16>(p, rows, pdl != 0, stream);
}
