// What stands between a model's logits and the probabilities that words are drawn from or drafts verified against: penalties for repeated words, biases, temperature,
// a grammar's mask.  Of a row with history h (the first of it a prompt), word w, n(w) its times behind the prompt:
//
//   z = z / repetition (z > 0) or z * repetition, where w is in h;   z -= frequency * n(w) + presence, where n(w) > 0
//   z += its biases, one after the other;   z /= temperature;   -inf, where the mask has no bit for w
//
// A CTA has a piece of a row's vocabulary, with a counter in shared memory for each word: how often it came, whether it is in the history, whether there is a bias.  Every CTA goes
// over the whole history and counts the words of its piece by atomics of its own shared memory: whole numbers, which add up the same in every order.  (With the history
// shared out among the CTAs of a cluster, and counts sent to the piece's owner: 52 us where this takes 28, 117 rows behind up to 9000 words, of which most are
// frequent ones that one CTA owns.)  Where 128 words are one it is counted once, so that a history of one word does not queue up.  The logits' first loads are
// on their way meanwhile.
//
// Few words of a piece are marked, mostly.  Whoever marks a word first puts it on a list; the piece is written as if there were none, and the marked words once more behind that.
// (With penalties worked out at every word, which costs three times the instructions of the rest, 64 rows of 128256 took 20 us instead of 18.)  Where
// the list is too long for shared memory that is done all the same.  Biases of a piece stand in a second list, in their order; of one that is too long for it the words go over the
// row's own.
#include "paged.cuh"

#include <climits>
#include <type_traits>

namespace zl {

constexpr int kAlThreads = 256, kAlAhead = 4, kAlList = 512;

// A counter: whether the word is in the history, whether there is a bias, how often it came behind the prompt.  16 bits where histories are short enough, two to a word of 32.
template <typename C>
struct AlCounter {
    static constexpr int kBits = 8 * sizeof(C), kEach = 32 / kBits;
    static constexpr uint32_t kSeen = 1u << (kBits - 1), kBias = 1u << (kBits - 2), kCount = kBias - 1;
    // before the change
    static __device__ __forceinline__ uint32_t add(uint32_t* c, int i, uint32_t n) { return (C)(atomicAdd(c + i / kEach, n << (i % kEach * kBits)) >> (i % kEach * kBits)); }
    static __device__ __forceinline__ uint32_t mark(uint32_t* c, int i, uint32_t bit) { return (C)(atomicOr(c + i / kEach, bit << (i % kEach * kBits)) >> (i % kEach * kBits)); }
};
constexpr int kAlShort = 0x3fff;

struct AdjustLogits {
    const void* in;
    void* out;
    long long ld_in, ld_out;
    const int32_t *tokens, *token_seq, *token_lens, *prompt_lens, *bias_starts, *bias_words, *mask, *mask_row;
    const float *repetition, *frequency, *presence, *bias, *temperature;
    long long ld_tokens, ld_mask;
    int seqs, longest, n_bias, masks, vocab, pieces, piece, in_place, room;   // room: of the list of marked words
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
__global__ void __launch_bounds__(kAlThreads, 4) k_adjust_logits(const AdjustLogits p) {
    using Counter = AlCounter<C>;
    constexpr int kAhead = VEC == 1 ? 8 : 4, kStep = kAlThreads * VEC, kEach = kAlList / kAlThreads;
    extern __shared__ __align__(16) uint32_t al_count[];
    constexpr int kHave = kEach * kAlThreads / 32;
    __shared__ int s_words[kAlList], s_have[kHave];
    __shared__ float s_bias[kAlList];
    __shared__ int s_marks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r = p.by_pieces((int)blockIdx.x), lo = min(((int)blockIdx.x - r * p.pieces) * p.piece, p.vocab), hi = min(lo + p.piece, p.vocab);
    uint16_t* s_marked = reinterpret_cast<uint16_t*>(al_count + (p.piece + 8) / Counter::kEach);
    TI* s_was = reinterpret_cast<TI*>(s_marked + p.room);   // their logits, where out is in
    const bool counts = p.tokens != nullptr, marks = counts || p.bias_starts;
    const TI* in = static_cast<const TI*>(p.in) + (long long)r * p.ld_in;
    TO* out = static_cast<TO*>(p.out) + (long long)r * p.ld_out;
    // Vectors stand on borders of 16 bytes: the first one begins up to VEC - 1 words before the piece
    const int base = lo - (int)(reinterpret_cast<uintptr_t>(in + lo) / sizeof(TI) % VEC);
    if (marks) {
        if (tid == 0) s_marks = 0;
        for (int i = tid * 4; i < (hi - base + Counter::kEach - 1) / Counter::kEach; i += kAlThreads * 4) *reinterpret_cast<uint4*>(al_count + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    pdl_trigger();
    pdl_wait();
    TI x[kAhead][VEC];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * kStep;
            if (i >= lo && i + VEC <= hi) al_load(x[u], in + i);
            else
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (i + e >= lo && i + e < hi) x[u][e] = in[i + e];
        }
    };
    const int start = base + tid * VEC;
    fetch(start);
    int first = 0, last = 0;   // of the biases
    // Clamped at both ends before anything is added to them: a start near the largest integer would wrap around, to places before the list.
    if (p.bias_starts) first = min(max(p.bias_starts[r], 0), p.n_bias), last = max(min(p.bias_starts[r + 1], p.n_bias), first);
    const int seq = !counts ? -1 : p.token_seq ? p.token_seq[r] : r, length = counts ? p.token_lens[r] : 0, prompt = p.prompt_lens ? p.prompt_lens[r] : 0;
    int mine[kEach];   // this thread's of the first ones, and what they are
    float mine_bias[kEach];
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
        const int i = first + u * kAlThreads + tid;
        mine[u] = -1, mine_bias[u] = 0.f;
        if (i < last) mine[u] = p.bias_words[i], mine_bias[u] = p.bias[i];
    }
    const float rep = p.repetition ? p.repetition[r] : 1.f, up = 1.f / rep, freq = p.frequency ? p.frequency[r] : 0.f, pres = p.presence ? p.presence[r] : 0.f;
    const float given = p.temperature ? p.temperature[r] : 0.f, heat = given >= 1.17549435e-38f ? given : 1.f, inv = 1.f / heat;
    // z / by: by the reciprocal and one correction of what is too much (Markstein 1990), which is a number where z, the divisor and the quotient are; -0 stays -0
    auto quotient = [](float z, float by, float inverse) {
        const float q = z * inverse, over = fmaf(q, by, -z);
        return fabsf(over) < INFINITY ? fmaf(-over, inverse, q) : q;
    };
    auto cooled = [&](float z) { return quotient(z, heat, inv); };
    const int mask_row = !p.mask ? -1 : p.mask_row ? p.mask_row[r] : r;
    const int32_t* mask = mask_row >= 0 && mask_row < p.masks ? p.mask + (long long)mask_row * p.ld_mask : nullptr;
    // a counter before it was changed: a word that had no mark goes on the list
    auto note = [&](bool is_first, int off) {
        const unsigned firsts = __ballot_sync(0xffffffffu, is_first);
        if (firsts == 0) return;
        int to = 0;
        if (lane == 0) to = atomicAdd(&s_marks, __popc(firsts));
        to = __shfl_sync(0xffffffffu, to, 0) + __popc(firsts & ((1u << lane) - 1u));
        if (is_first && to < p.room) s_marked[to] = (uint16_t)off;
    };
    if (counts) {
        const int n = seq >= 0 && seq < p.seqs ? min(length, p.longest) : 0;
        const int32_t* words = p.tokens + (long long)max(seq, 0) * p.ld_tokens;
        const unsigned from = (unsigned)(lo - base), size = (unsigned)(hi - lo);
        auto go = [&](int i, const int end, auto behind) {   // words i .. end - 1
            constexpr bool kBehind = decltype(behind)::value;
            for (i += tid; i - lane < end; i += kAlAhead * kAlThreads) {
                int off[kAlAhead];
#pragma unroll
                for (int u = 0; u < kAlAhead; ++u) off[u] = i + u * kAlThreads < end ? words[i + u * kAlThreads] - base : -1 - base;
                const int of_first = __shfl_sync(0xffffffffu, off[0], 0);
                bool one = true;
#pragma unroll
                for (int u = 0; u < kAlAhead; ++u) one &= off[u] == of_first;
                if (__all_sync(0xffffffffu, one)) {
                    uint32_t before = 1;
                    if (lane == 0 && (unsigned)off[0] - from < size) before = kBehind ? Counter::add(al_count, off[0], 32u * kAlAhead) : Counter::mark(al_count, off[0], Counter::kSeen);
                    note(before == 0, off[0]);
                    continue;
                }
#pragma unroll
                for (int u = 0; u < kAlAhead; ++u) {
                    uint32_t before = 1;
                    if ((unsigned)off[u] - from < size) before = kBehind ? Counter::add(al_count, off[u], 1u) : Counter::mark(al_count, off[u], Counter::kSeen);
                    note(before == 0, off[u]);
                }
            }
        };
        const int middle = min(max(prompt, 0), n);
        if (middle > 0) go(0, middle, std::false_type{});
        if (n > middle) go(middle, n, std::true_type{});
    }
    int listed = -1;   // -1: the row's own list
    if (last - first <= kAlList) {
        listed = 0;
        if (first < last) {
            unsigned here[kEach];
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                here[u] = __ballot_sync(0xffffffffu, mine[u] >= lo && mine[u] < hi);
                if (lane == 0) s_have[u * (kAlThreads / 32) + warp] = __popc(here[u]);
            }
            __syncthreads();
            int at[kEach] = {};
            for (int w = 0; w < kHave; ++w) {
                const int n = s_have[w];
#pragma unroll
                for (int u = 0; u < kEach; ++u)
                    if (w < u * (kAlThreads / 32) + warp) at[u] += n;
                listed += n;
            }
#pragma unroll
            for (int u = 0; u < kEach; ++u)
                if (here[u] >> lane & 1u) {
                    const int to = at[u] + __popc(here[u] & ((1u << lane) - 1u));
                    s_words[to] = mine[u], s_bias[to] = mine_bias[u];
                }
        }
    }
    for (int i0 = first + warp * 32, u = 0; i0 < last; i0 += kAlThreads, ++u) {
        const int word = u == 0 ? mine[0] : i0 + lane < last ? p.bias_words[i0 + lane] : -1, off = word - base;
        const bool is = word >= lo && word < hi;
        uint32_t before = 1;
        if (is) before = Counter::mark(al_count, off, Counter::kBias);
        note(before == 0, off);
    }
    if (marks) __syncthreads();
    const C* marked = reinterpret_cast<const C*>(al_count);
    auto adjusted = [&](float z, uint32_t mark, int word) {
        const uint32_t n = mark & Counter::kCount;
        if (mark & (Counter::kCount | Counter::kSeen)) z = z > 0.f ? (fabsf(up) < INFINITY ? quotient(z, rep, up) : z / rep) : z * rep;
        if (n) z -= fmaf(freq, (float)n, pres);
        if (mark & Counter::kBias) {
            if (listed >= 0) {
#pragma unroll 8
                for (int b = 0; b < listed; ++b)
                    if (s_words[b] == word) z += s_bias[b];
            } else {
                for (int b = first; b < last; ++b)
                    if (p.bias_words[b] == word) z += p.bias[b];
            }
        }
        return z;
    };
    const int some = marks ? s_marks : 0;
    auto ends = [&](float z, int word) { return from_f32<TO>(!mask || ((uint32_t)mask[word >> 5] >> (word & 31) & 1u) ? cooled(z) : -INFINITY); };
    if (some > p.room) {   // word by word
        for (int i = lo + tid; i < hi; i += kAlThreads) {
            const float z = to_f32<TI>(in[i]);
            const uint32_t mark = marked[i - base];
            out[i] = ends(mark ? adjusted(z, mark, i) : z, i);
        }
        return;
    }
    // Logits of marked words as they are: the first of each thread's in registers, on their way while the piece is written
    constexpr int kWas = 6;
    TI was[kWas];
#pragma unroll
    for (int u = 0; u < kWas; ++u)
        if (u * kAlThreads + tid < some) was[u] = in[base + s_marked[u * kAlThreads + tid]];
    if (p.in_place && some) {
        for (int i = kWas * kAlThreads + tid; i < some; i += kAlThreads) s_was[i] = in[base + s_marked[i]];
        __syncthreads();
    }
    for (int i0 = start; i0 < hi; i0 += kAhead * kStep) {
        if (i0 != start) fetch(i0);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * kStep;
            if (i >= hi) break;
            uint32_t allowed = 0xffffffffu;
            if (mask) {   // bits of words i .. i + VEC - 1; behind the row's end there may be none
                const int w = max(i, 0) >> 5;
                allowed = i < 0 ? (uint32_t)mask[0] << -i : (uint32_t)mask[w] >> (i & 31);
                if (VEC > 1 && (i & 31) + VEC > 32 && i > 0 && (w + 1) * 32 < hi) allowed |= (uint32_t)mask[w + 1] << (32 - (i & 31));
            }
            float z[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) z[e] = to_f32<TI>(x[u][e]);
            TO y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[e] = from_f32<TO>(allowed >> e & 1u ? cooled(z[e]) : -INFINITY);
            if constexpr (VEC == 1) out[i] = y[0];
            else if (i < lo || i + VEC > hi)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if (i + e >= lo && i + e < hi) out[i + e] = y[e];
                }
            else
#pragma unroll
                for (int e = 0; e < VEC * (int)sizeof(TO); e += 16) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out + i) + e) = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(y) + e);
        }
    }
    if (some == 0) return;
    __syncthreads();
    auto again = [&](int i, TI x) {
        const int off = s_marked[i], word = base + off;
        out[word] = ends(adjusted(to_f32<TI>(x), marked[off], word), word);
    };
#pragma unroll
    for (int u = 0; u < kWas; ++u)
        if (u * kAlThreads + tid < some) again(u * kAlThreads + tid, was[u]);
    for (int i = kWas * kAlThreads + tid; i < some; i += kAlThreads) again(i, p.in_place ? s_was[i] : in[base + s_marked[i]]);
}

constexpr int kAlMaxBytes = 34 * 1024, kAlMaxList = 16 * 1024;   // of a piece's counters, of words that are marked

template <typename TI, typename TO, typename C>
static int adjust_logits(AdjustLogits p, int rows, bool pdl, zl_stream_t stream) {
    // 16 bytes at a time where the borders of 16 bytes of a row lie at the same words in both; 117 rows of 50257 30 us word by word, 26 so, when the rest was otherwise
    constexpr int kVec = 16 / sizeof(TI), kOut = 16 / sizeof(TO);
    const long long ahead = (long long)(reinterpret_cast<uintptr_t>(p.in) / sizeof(TI) % kVec) - (long long)(reinterpret_cast<uintptr_t>(p.out) / sizeof(TO) % kOut);
    const bool wide = ahead % kOut == 0 && (p.ld_in - p.ld_out) % kOut == 0 && reinterpret_cast<uintptr_t>(p.in) % sizeof(TI) == 0 && reinterpret_cast<uintptr_t>(p.out) % sizeof(TO) == 0;
    // counters, with words before the piece; no more marked words than the piece has, or the history and the biases
    const long long marks = (long long)p.longest + p.n_bias;
    p.room = (int)(marks < p.piece ? marks : p.piece);
    if (p.room > kAlMaxList / (p.in_place ? 3 : 1)) p.room = kAlMaxList / (p.in_place ? 3 : 1);
    p.room = (p.room + 7) / 8 * 8;
    const size_t smem = p.tokens || p.bias_starts ? (size_t)(p.piece + 8) * sizeof(C) + p.room * (2 + (p.in_place ? sizeof(TI) : 0)) : 0;
    const auto kernel = wide ? k_adjust_logits<TI, TO, C, kVec> : k_adjust_logits<TI, TO, C, 1>;
    if (smem > 32 * 1024) {
        static bool done[2][64] = {};
        int dev = 0;
        cudaGetDevice(&dev);
        if (dev < 0 || dev >= 64 || !done[wide][dev]) {
            ZL_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kAlMaxBytes + 2 * kAlMaxList + 256));
            if (dev >= 0 && dev < 64) done[wide][dev] = true;
        }
    }
    ZL_CHECK_CUDA(launch(kernel, dim3((unsigned)rows * p.pieces), dim3(kAlThreads), smem, stream, pdl, p));
    return ZL_OK;
}

// The number of pieces: the fewest cycles of the SM that has the most, of 26 for 100 words (the bytes), 12 for 100 words of history and 300 for a CTA, from three CTAs an SM on.  A piece
// has 1024 words or more, and counters that leave room for four CTAs (three where the list of marked words takes all that it may).  us by the number of pieces, 117 rows of 50257 behind up to 9000 words: 3 37, 4 43, 5 28 (taken), 6 32, 9 36;
// 64 rows of 128256 behind up to 4000: 4 21, 6 20, 9 18 (taken).  CTAs of 1024 threads, of which one piece a row is best: 32 and 19.
// Against the best of up to 18 numbers of pieces, over rows of 1 to 512, vocabularies of 8000 to 152064 and histories of none to 16000 words (bf16 to fp32, 124 calls, in a graph): within 5 %
// for 89 of them, within 20 % for all but two: 8 rows of 50257 without histories 4.2 instead of 3.2, 64 of 152064 14.5 instead of 11.3.
static int al_pieces(int rows, int vocab, int longest, int counter) {
    const int least = (int)(((long long)vocab * counter - 1) / (kAlMaxBytes - 128)) + 1, sms = device_sm_count();
    const int most = vocab / 1024 < least ? least : vocab / 1024 < least + 256 ? vocab / 1024 : least + 256;
    int best = least;
    double cost = 0.0;
    for (int n = least; n <= most; ++n) {
        const long long ctas = ((long long)rows * n + sms - 1) / sms;
        if (ctas < 3 && n < most) continue;
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
    ZL_CHECK_SUPPORTED(!bias_starts || n_bias <= INT_MAX - 1024);   // a CTA's look ahead from the list's end is counted in 32 bits
    ZL_CHECK_ARG(!mask || (masks > 0 && ld_mask >= (vocab - 1) / 32 + 1 && (mask_row || masks >= rows)));
    ZL_CHECK_SUPPORTED(vocab <= 1 << 24 && longest < 1 << 23 && (out_dtype == dtype || out_dtype == ZL_F32) && (dtype == ZL_F32 || dtype == ZL_F16 || dtype == ZL_BF16));
    AdjustLogits p = {logits, out, ld_logits, ld_out, tokens, token_seq, token_lens, prompt_lens, bias_starts, bias_words, mask, mask_row,
                      repetition, frequency, presence, bias, temperature, ld_tokens, ld_mask, seqs, tokens ? longest : 0, bias_starts ? n_bias : 0, masks, vocab};
    // Out may be logits itself, or lie beside it in the same rows; else a word could be read after another one was written over it
    const long long size = dtype == ZL_F32 ? 4 : 2, out_size = out_dtype == ZL_F32 ? 4 : 2, ahead = (long long)(reinterpret_cast<uintptr_t>(out) - reinterpret_cast<uintptr_t>(logits));
    const long long step = rows > 1 ? ld_logits * size : 0, out_step = rows > 1 ? ld_out * out_size : 0;
    const bool apart = ahead >= (rows - 1) * step + vocab * size || -ahead >= (rows - 1) * out_step + vocab * out_size;
    if (!apart) {
        const bool same = ahead == 0 && step == out_step && size == out_size && dtype == out_dtype;
        const long long beside = step > 0 && step == out_step ? (ahead % step + step) % step : 0;
        ZL_CHECK_SUPPORTED(same || (beside >= vocab * size && step - beside >= vocab * out_size));
    }
    p.in_place = !apart;
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
