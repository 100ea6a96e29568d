// What stands between a model's logits and the probabilities that words are drawn from or drafts verified against: penalties for repeated words, biases, temperature,
// a grammar's mask.  Of a row with history h (the first of it a prompt), word w, n(w) its times behind the prompt:
//
//   z = z * (1 / repetition) (z > 0) or z * repetition, where w is in h;   z -= frequency * n(w) + presence, where n(w) > 0
//   z += its biases, one after the other;   z *= 1 / temperature;   -inf, where the mask has no bit for w
//
// A CTA has a piece of a row's vocabulary, with a counter in shared memory for each word: how often it came, whether it is in the history, whether there is a bias.  Every CTA goes
// over the whole history and counts the words of its piece by atomics of its own shared memory: whole numbers, which add up the same in every order.  (With the history
// shared out among the CTAs of a cluster, and counts sent to the piece's owner: 52 us where this takes %s, 117 rows behind 9000 words, of which most are
// frequent ones that one CTA owns.)  A warp whose 32 words are one counts it once, so that a history of one word does not queue up.  The logits' first loads are
// on their way meanwhile.
//
// Biases of a piece stand in a list, in their order, with their words' logits as they were; once the piece is written a thread for each word writes those
// again.  (A search of the list at every marked word took most of the time: 300 biases a row.)  Of a list that is too long for this, each marked word
// goes over the row's own list.
#include "paged.cuh"

namespace zl {

constexpr int kAlThreads = 512, kAlAhead = 4;

// A counter: whether the word is in the history, whether there is a bias, how often it came behind the prompt.  16 bits where histories are short enough.
template <typename C>
struct AlCounter {
    static constexpr int kBits = 8 * sizeof(C);
    static constexpr uint32_t kSeen = 1u << (kBits - 1), kBias = 1u << (kBits - 2), kCount = kBias - 1, kEach = 32 / kBits;   // of 32 bits
    static __device__ __forceinline__ uint32_t* at(uint32_t* words, int i) { return words + i / kEach; }
    static __device__ __forceinline__ uint32_t shifted(uint32_t x, int i) { return x << (i % kEach * kBits); }
};
constexpr int kAlShort = 0x3fff;

struct AdjustLogits {
    const void* in;
    void* out;
    long long ld_in, ld_out;
    const int32_t *tokens, *token_seq, *token_lens, *prompt_lens, *bias_starts, *bias_words, *mask, *mask_row;
    const float *repetition, *frequency, *presence, *bias, *temperature;
    long long ld_tokens, ld_mask;
    int seqs, longest, n_bias, masks, vocab, pieces, piece;
    PagedDivisor by_pieces;
};

template <typename TI, int VEC>
__device__ __forceinline__ void al_load(TI (&v)[VEC], const TI* at) {
    if constexpr (VEC * sizeof(TI) == 16) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(at);
    else
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = at[i];
}

// grid: pieces of rows; dynamic shared memory: a counter for each of the piece's words, where there is a history or a bias
template <typename TI, typename TO, typename C, int VEC>
__global__ void __launch_bounds__(kAlThreads) k_adjust_logits(const AdjustLogits p) {
    using Counter = AlCounter<C>;
    constexpr int kAhead = VEC == 1 ? 8 : 2, kStep = kAlThreads * VEC;
    extern __shared__ __align__(16) uint32_t al_count[];
    __shared__ int s_words[kAlThreads], s_have[kAlThreads / 32];
    __shared__ float s_bias[kAlThreads], s_logit[kAlThreads];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r = p.by_pieces((int)blockIdx.x), lo = min(((int)blockIdx.x - r * p.pieces) * p.piece, p.vocab), hi = min(lo + p.piece, p.vocab);
    const bool counts = p.tokens != nullptr, marks = counts || p.bias_starts;
    if (marks) {
        for (int i = tid * 4; i < (hi - lo + (int)Counter::kEach - 1) / (int)Counter::kEach; i += kAlThreads * 4) *reinterpret_cast<uint4*>(al_count + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    pdl_trigger();
    pdl_wait();
    const TI* in = static_cast<const TI*>(p.in) + (long long)r * p.ld_in;
    TO* out = static_cast<TO*>(p.out) + (long long)r * p.ld_out;
    TI x[kAhead][VEC];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (i0 + u * kStep < hi) al_load(x[u], in + i0 + u * kStep);
    };
    const int start = lo + tid * VEC;
    fetch(start);
    int first = 0, last = 0;   // of the biases
    if (p.bias_starts) first = max(p.bias_starts[r], 0), last = min(p.bias_starts[r + 1], p.n_bias);
    const int mine = first + tid < last ? p.bias_words[first + tid] : -1;   // this thread's of the first ones
    const float rep = p.repetition ? p.repetition[r] : 1.f, up = 1.f / rep, freq = p.frequency ? p.frequency[r] : 0.f, pres = p.presence ? p.presence[r] : 0.f;
    const float heat = p.temperature ? p.temperature[r] : 0.f, inv = heat >= 1.17549435e-38f ? 1.f / heat : 1.f;
    const int mask_row = !p.mask ? -1 : p.mask_row ? p.mask_row[r] : r;
    const int32_t* mask = mask_row >= 0 && mask_row < p.masks ? p.mask + (long long)mask_row * p.ld_mask : nullptr;
    if (counts) {
        const int seq = p.token_seq ? p.token_seq[r] : r, n = seq >= 0 && seq < p.seqs ? min(p.token_lens[r], p.longest) : 0, prompt = p.prompt_lens ? p.prompt_lens[r] : 0;
        const int32_t* words = p.tokens + (long long)max(seq, 0) * p.ld_tokens;
        for (int i0 = tid; i0 - lane < n; i0 += kAlAhead * kAlThreads) {
            int word[kAlAhead];
#pragma unroll
            for (int u = 0; u < kAlAhead; ++u) word[u] = i0 + u * kAlThreads < n ? words[i0 + u * kAlThreads] : -1;
#pragma unroll
            for (int u = 0; u < kAlAhead; ++u) {
                const int off = word[u] - lo;
                const bool is = word[u] >= lo && word[u] < hi, behind = i0 + u * kAlThreads >= prompt;
                if (!__any_sync(0xffffffffu, is)) continue;
                const int key = is ? off << 1 | (int)behind : -1;
                const bool one = __all_sync(0xffffffffu, key == __shfl_sync(0xffffffffu, key, 0));
                if (is && (!one || lane == 0)) {
                    if (behind) atomicAdd(Counter::at(al_count, off), Counter::shifted(one ? 32u : 1u, off));
                    else atomicOr(Counter::at(al_count, off), Counter::shifted(Counter::kSeen, off));
                }
            }
        }
    }
    int listed = 0;
    if (first < last && last - first <= kAlThreads) {
        const bool is = mine >= lo && mine < hi;
        const unsigned here = __ballot_sync(0xffffffffu, is);
        if (lane == 0) s_have[warp] = __popc(here);
        __syncthreads();
        int at = __popc(here & ((1u << lane) - 1u));
        for (int w = 0; w < kAlThreads / 32; ++w) {
            const int n = s_have[w];
            if (w < warp) at += n;
            listed += n;
        }
        if (is) s_words[at] = mine, s_bias[at] = p.bias[first + tid], s_logit[at] = to_f32<TI>(in[mine]);
    } else {
        for (int i = first + tid; i < last; i += kAlThreads) {
            const int off = p.bias_words[i] - lo;
            if (off >= 0 && off < hi - lo) atomicOr(Counter::at(al_count, off), Counter::shifted(Counter::kBias, off));
        }
    }
    if (marks) __syncthreads();
    const C* marked = reinterpret_cast<const C*>(al_count);
    auto penalised = [&](float z, uint32_t mark) {
        const uint32_t n = mark & Counter::kCount;
        if (mark & (Counter::kCount | Counter::kSeen)) z *= z > 0.f ? up : rep;
        return n ? z - fmaf(freq, (float)n, pres) : z;
    };
    for (int i0 = start; i0 < hi; i0 += kAhead * kStep) {
        if (i0 != start) fetch(i0);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * kStep;
            if (i >= hi) break;
            const uint32_t allowed = mask ? (uint32_t)mask[i >> 5] >> (i & 31) : 0xffffffffu;
            float z[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) z[e] = to_f32<TI>(x[u][e]);
            if (marks) {
                C mark[VEC];
                bool any = true;
                if constexpr (VEC * sizeof(C) >= 8) {
                    uint2 w[VEC * sizeof(C) / 8];
                    any = false;
#pragma unroll
                    for (int e = 0; e < VEC * (int)sizeof(C) / 8; ++e) {
                        w[e] = *reinterpret_cast<const uint2*>(marked + (i - lo) + e * 8 / (int)sizeof(C));
                        any |= (w[e].x | w[e].y) != 0;
                        *reinterpret_cast<uint2*>(mark + e * 8 / (int)sizeof(C)) = w[e];
                    }
                } else {
                    mark[0] = marked[i - lo];
                }
                if (any)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        z[e] = penalised(z[e], mark[e]);
                        if (mark[e] & Counter::kBias)
                            for (int b = first; b < last; ++b)
                                if (p.bias_words[b] == i + e) z[e] += p.bias[b];
                    }
            }
            TO y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[e] = from_f32<TO>(allowed >> e & 1u ? z[e] * inv : -INFINITY);
            if constexpr (VEC == 1) out[i] = y[0];
            else
#pragma unroll
                for (int e = 0; e < VEC * (int)sizeof(TO); e += 16) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out + i) + e) = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(y) + e);
        }
    }
    if (listed == 0) return;
    __syncthreads();
    if (tid >= listed) return;
    const int word = s_words[tid];
    bool again = false;
    for (int b = 0; b < tid; ++b) again |= s_words[b] == word;
    if (again) return;   // the first one sees to it
    float z = penalised(s_logit[tid], marked[word - lo]) + s_bias[tid];
    for (int b = tid + 1; b < listed; ++b)
        if (s_words[b] == word) z += s_bias[b];
    const bool allowed = !mask || ((uint32_t)mask[word >> 5] >> (word & 31) & 1u);
    out[word] = from_f32<TO>(allowed ? z * inv : -INFINITY);
}

template <typename TI, typename TO, typename C>
static int adjust_logits(const AdjustLogits& p, int rows, bool pdl, zl_stream_t stream) {
    // whole 16 bytes where rows and pitches allow it
    constexpr int kVec = 16 / sizeof(TI);
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.in) | reinterpret_cast<uintptr_t>(p.out);
    const bool wide = at % 16 == 0 && p.vocab % kVec == 0 && p.ld_in * sizeof(TI) % 16 == 0 && p.ld_out * sizeof(TO) % 16 == 0;
    const size_t smem = p.tokens || p.bias_starts ? (size_t)p.piece * sizeof(C) : 0;
    ZL_CHECK_CUDA(launch(wide ? k_adjust_logits<TI, TO, C, kVec> : k_adjust_logits<TI, TO, C, 1>, dim3((unsigned)rows * p.pieces), dim3(kAlThreads), smem, stream, pdl, p));
    return ZL_OK;
}

// The number of pieces: the fewest cycles of the SM that has the most, of 26 for 100 words (the bytes), 12 for 100 words of history and 300 for a CTA.  A piece has up to 40 KB of counters,
// so that an SM holds four, and 1024 words or more.  117 rows of 50257 behind 9000: 5, 64 rows of 128256 behind 4000: 9, one row of 32000: 31.
static int al_pieces(int rows, int vocab, int longest, int counter) {
    const int least = (int)(((long long)vocab * counter - 1) / (40 * 1024 - 64)) + 1, most = vocab / 1024 > least ? vocab / 1024 : least, sms = device_sm_count();
    int best = least;
    double cost = 0.0;
    for (int n = least; n <= most && n <= least + 256; ++n) {
        const long long ctas = ((long long)rows * n + sms - 1) / sms;
        if (ctas < 3 && n < most) continue;   // for what an SM has in flight
        const double x = (double)ctas * (0.26 * vocab / n + 0.12 * longest + 300.0);
        if (cost == 0.0 || x < cost) cost = x, best = n;
    }
    return best;
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
    ZL_CHECK_SUPPORTED(vocab <= 1 << 24 && longest <= 1 << 29 && (out_dtype == dtype || out_dtype == ZL_F32) && (dtype == ZL_F32 || dtype == ZL_F16 || dtype == ZL_BF16));
    AdjustLogits p = {logits, out, ld_logits, ld_out, tokens, token_seq, token_lens, prompt_lens, bias_starts, bias_words, mask, mask_row,
                      repetition, frequency, presence, bias, temperature, ld_tokens, ld_mask, seqs, tokens ? longest : 0, n_bias, masks, vocab};
    const bool counts16 = p.longest <= kAlShort;
    p.pieces = al_pieces(rows, vocab, p.longest, counts16 ? 2 : 4);
    p.piece = (((vocab - 1) / p.pieces + 1) + 31) / 32 * 32;
    p.by_pieces = paged_divisor(p.pieces);
    ZL_CHECK_SUPPORTED((long long)rows * p.pieces < 1ll << 31);
    const bool dep = pdl != 0;
    auto with = [&](auto counter) {
        using C = decltype(counter);
        if (dtype == ZL_F32) return adjust_logits<float, float, C>(p, rows, dep, stream);
        if (dtype == ZL_F16) return out_dtype == ZL_F32 ? adjust_logits<__half, float, C>(p, rows, dep, stream) : adjust_logits<__half, __half, C>(p, rows, dep, stream);
        return out_dtype == ZL_F32 ? adjust_logits<__nv_bfloat16, float, C>(p, rows, dep, stream)
                                   : adjust_logits<__nv_bfloat16, __nv_bfloat16, C>(p, rows, dep, stream);
    };
    return counts16 ? with(uint16_t{}) : with(uint32_t{});
}
