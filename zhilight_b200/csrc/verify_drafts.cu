// Verification of drafted tokens against the target's probabilities from given random numbers (the rejection scheme published as speculative
// sampling by Leviathan et al. and Chen et al., 2023): draft i with word x is taken while u_i q_i(x) < p_i(x).  At the first one refused the word comes
// from the weights max(p - q, 0) of that row, behind the last draft from p itself: the first index whose running sum passes u * (sum of all).
//
// Only that one row of p and q is read whole.  The CTAs of a cluster share the vocabulary, a warp has a run of neighbouring words: a pass for the sums
// of the warps, which every CTA gets from the others' shared memory, then the CTA that has the word's run goes over that run once more.
// Differences, products and sums are in 64 bits: products of two 32-bit numbers are exact there, sums of probabilities above 2^-29 too, and
// a tie falls as the formula says.  A sequence whose drafts were all taken reads no row of q: of 64 sequences with up to 5 drafts 21 to 24 refuse one, 44 to 45 MB for
// 128256 words.  15.4 us in a graph with the rows in L2 (2.9 TB/s), 17 a call, 18 under ncu with cold caches (2.5 TB/s; DRAM 31 %, SMs 28 % busy): bound by neither, but by a chain of
// three dependent loads, a pass behind them, the cluster's barrier and the run once more (6.9 us for one sequence of 32000 words), all CTAs in one wave.
// Eight warps of 16 loads ahead; 16 warps of 8, of which an SM holds three CTAs, took 21.5 us where these took 15.4, of 16 23.1; four CTAs of 32 registers 19.5.
#include "paged.cuh"
#include "tc2_common.cuh"

#include <climits>

namespace zl {

constexpr int kVdWarps = 8, kVdMaxCluster = 8, kVdAhead = 16;

constexpr int kVdEach = kVdMaxCluster * kVdWarps / 32;   // sums of runs that a lane looks at

__device__ __forceinline__ double vd_scan(double v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}

// the weight of a word; what is not finite or not positive counts as none
__device__ __forceinline__ double vd_weight(float a, float q) { return a > q && a < INFINITY && q > -INFINITY ? (double)a - (double)q : 0.0; }

// This lane's share of the weights of lo .. hi - 1: target less draft (TWO), or target alone, less one at `skip`
template <bool TWO>
__device__ __forceinline__ double vd_sum(const float* __restrict__ tr, const float* __restrict__ dr, int lo, int hi, int skip) {
    double s[2] = {0.0, 0.0};
    int i = lo + (threadIdx.x & 31);
    float a[kVdAhead], q[kVdAhead];
    for (; i + 32 * (kVdAhead - 1) < hi; i += 32 * kVdAhead) {
#pragma unroll
        for (int u = 0; u < kVdAhead; ++u) {
            a[u] = tr[i + 32 * u];
            if (TWO) q[u] = dr[i + 32 * u];
        }
#pragma unroll
        for (int u = 0; u < kVdAhead; ++u) s[u & 1] += vd_weight(a[u], TWO ? q[u] : i + 32 * u == skip ? 1.f : 0.f);
    }
#pragma unroll
    for (int u = 0; u < kVdAhead; ++u) {
        a[u] = i + 32 * u < hi ? tr[i + 32 * u] : 0.f;
        if (TWO) q[u] = i + 32 * u < hi ? dr[i + 32 * u] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kVdAhead; ++u) s[u & 1] += vd_weight(a[u], TWO ? q[u] : i + 32 * u == skip ? 1.f : 0.f);
    return s[0] + s[1];
}

struct VerifyDrafts {
    const float *target, *draft;
    long long t_seq, t_row, d_seq, d_row;
    const int32_t *drafted, *count;
    const float *accept, *sample;
    int32_t *accepted, *tokens;
    int k, vocab;
};

// grid (CTAs of a sequence, sequences), a cluster along x
__global__ void __launch_bounds__(kVdWarps * 32) k_verify_drafts(const VerifyDrafts p) {
    __shared__ double part[kVdMaxCluster][kVdWarps];
    __shared__ double s_sum[kVdWarps];
    __shared__ int s_taken, s_count, s_first[kVdWarps], s_last[kVdWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.y, ctas = gridDim.x, cta = blockIdx.x;
    if (ctas > 1) cluster_arrive();   // every CTA runs before another one stores into it
    pdl_trigger();
    pdl_wait();
    if (warp == 0) {
        int taken = 0, n = p.k;
        for (int i0 = 0; i0 < n; i0 += 32) {
            const int i = i0 + lane;
            int x = -1;
            float u = 0.f;
            if (i < n) x = p.drafted[(size_t)b * p.k + i], u = p.accept[(size_t)b * p.k + i];
            if (i0 == 0 && p.count) n = min(max(p.count[b], 0), p.k);   // beside the two above
            bool ok = false;
            if (i < n && (unsigned)x < (unsigned)p.vocab) {
                const double q = p.draft ? (double)p.draft[b * p.d_seq + i * p.d_row + x] : 1.0;
                ok = (double)u * q < (double)p.target[b * p.t_seq + i * p.t_row + x];
            }
            const unsigned m = __ballot_sync(0xffffffffu, ok);
            taken += m == 0xffffffffu ? 32 : __ffs(~m) - 1;
            if (m != 0xffffffffu) break;
        }
        if (lane == 0) s_taken = min(taken, n), s_count = n;
    }
    __syncthreads();
    const int taken = s_taken;
    const bool refused = taken < s_count;
    const float* tr = p.target + b * p.t_seq + taken * p.t_row;
    const float* dr = refused && p.draft ? p.draft + b * p.d_seq + taken * p.d_row : nullptr;
    const int skip = refused && !p.draft ? p.drafted[(size_t)b * p.k + taken] : -1;   // a draft without probabilities has all of its own on one word
    // this warp's run
    const int run = cdiv(p.vocab, ctas * kVdWarps), lo = min((cta * kVdWarps + warp) * run, p.vocab), hi = min(lo + run, p.vocab);
    double total = 0.0, below = 0.0, each[kVdEach];
    bool plain = !refused;
    if (ctas > 1) cluster_wait();
    for (;;) {
        const double sum = plain || !dr ? vd_sum<false>(tr, nullptr, lo, hi, plain ? -1 : skip) : vd_sum<true>(tr, dr, lo, hi, -1);
        double mine = sum;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (ctas > 1) {
            if (lane < ctas) {
                const uint32_t at = cluster_map(smem_u32(&part[cta][warp]), (uint32_t)lane);
                asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(mine) : "memory");
            }
            cluster_sync_all();
        } else {
            if (lane == 0) part[0][warp] = mine;
            __syncthreads();
        }
        // sums of the runs up to and with this lane's, in order: up to four runs a lane
#pragma unroll
        for (int u = 0; u < kVdEach; ++u) {
            const int e = lane * kVdEach + u;
            each[u] = (u ? each[u - 1] : 0.0) + (e < ctas * kVdWarps ? part[e / kVdWarps][e % kVdWarps] : 0.0);
        }
        below = vd_scan(each[kVdEach - 1]);
        total = __shfl_sync(0xffffffffu, below, 31);
        below -= each[kVdEach - 1];   // for the places of the runs; which run has the word goes by these same numbers
        if (total > 0.0 || plain) break;
        plain = true;                    // nothing is left of the target: its own row decides
        if (ctas > 1) cluster_sync_all();   // the sums have been read
        else __syncthreads();
    }
    if (cta == 0 && tid <= p.k && tid != taken) p.tokens[(size_t)b * (p.k + 1) + tid] = tid < taken ? p.drafted[(size_t)b * p.k + tid] : -1;
    if (cta == 0)
        for (int i = tid + (int)blockDim.x; i <= p.k; i += blockDim.x)
            if (i != taken) p.tokens[(size_t)b * (p.k + 1) + i] = i < taken ? p.drafted[(size_t)b * p.k + i] : -1;
    if (cta == 0 && tid == 0) {
        p.accepted[b] = taken;
        if (!(total > 0.0)) p.tokens[(size_t)b * (p.k + 1) + taken] = -1;   // no word has any probability
    }
    if (!(total > 0.0)) return;
    // The warp whose run holds the word: the first whose running sum passes; behind them all (u of one, or sums that round apart) the last one that has
    // a weight.  Every warp knows all sums, so each tells by itself.
    const double goal = (double)p.sample[b] * total;
    int past = kVdEach, some = -1;   // of this lane's runs the first that passes, the last with a weight
#pragma unroll
    for (int u = kVdEach - 1; u >= 0; --u) {
        const bool weight = each[u] > (u ? each[u - 1] : 0.0);
        if (weight && below + each[u] > goal) past = u;
        if (weight && some < 0) some = u;
    }
    const unsigned passes = __ballot_sync(0xffffffffu, past < kVdEach), has = __ballot_sync(0xffffffffu, some >= 0);
    const int src = passes ? __ffs(passes) - 1 : 31 - __clz(has);
    const int owner = src * kVdEach + __shfl_sync(0xffffffffu, passes ? past : some, src);
    if (owner / kVdWarps != cta) return;
    // The run once more by the whole CTA: a piece of neighbouring words for every thread, then the words of the piece that passes.
    const int u0 = owner % kVdEach, from = min(owner * run, p.vocab), to = min(from + run, p.vocab), piece = cdiv(to - from, kVdWarps * 32);
    const int a = min(from + tid * piece, to), z = min(a + piece, to);
    auto weight_at = [&](int i) { return vd_weight(tr[i], plain ? 0.f : dr ? dr[i] : i == skip ? 1.f : 0.f); };
    double w = 0.0;
#pragma unroll 4
    for (int i = a; i < z; ++i) w += weight_at(i);
    const double up = vd_scan(w);
    if (lane == 31) s_sum[warp] = up;
    __syncthreads();
    double sum = lane < kVdWarps ? s_sum[lane] : 0.0;
    sum = vd_scan(sum) - sum;        // of the warps before
    sum = __shfl_sync(0xffffffffu, sum, warp) + __shfl_sync(0xffffffffu, below + (u0 ? each[u0 - 1] : 0.0), src);
    const unsigned here = __ballot_sync(0xffffffffu, w > 0.0 && sum + up > goal), any = __ballot_sync(0xffffffffu, w > 0.0);
    if (lane == 0) s_first[warp] = here ? tid + __ffs(here) - 1 : INT_MAX, s_last[warp] = any ? tid + 31 - __clz(any) : -1;
    __syncthreads();
    int first = __reduce_min_sync(0xffffffffu, lane < kVdWarps ? s_first[lane] : INT_MAX);
    const int back = __reduce_max_sync(0xffffffffu, lane < kVdWarps ? s_last[lane] : -1);
    if (first == INT_MAX) first = back;
    if (tid != first) return;
    int word = -1;
    sum += up - w;
    for (int i = a; i < z; ++i) {
        const double x = weight_at(i);
        sum += x;
        if (x > 0.0) word = i;
        if (x > 0.0 && sum > goal) break;
    }
    p.tokens[(size_t)b * (p.k + 1) + taken] = word;
}

}  // namespace zl

using namespace zl;

extern "C" int zl_verify_drafts(const float* target, long long target_seq, long long target_row, const float* draft, long long draft_seq,
                                long long draft_row, const int32_t* drafted, const float* accept, const float* sample, const int32_t* count,
                                int32_t* accepted, int32_t* tokens, int seqs, int drafts, int vocab, int pdl, zl_stream_t stream) {
    ZL_CHECK_ARG(target && sample && accepted && tokens && seqs > 0 && drafts >= 0 && vocab > 0);
    ZL_CHECK_ARG(drafts == 0 || (drafted && accept));
    ZL_CHECK_ARG(target_seq >= 0 && target_row >= 0 && draft_seq >= 0 && draft_row >= 0);
    ZL_CHECK_SUPPORTED(vocab <= 1 << 30 && seqs <= 65535);
    const VerifyDrafts p = {target, drafts ? draft : nullptr, target_seq, target_row, draft_seq, draft_row, drafted, count, accept, sample, accepted, tokens, drafts, vocab};
    int ctas = 1;
    while (ctas < kVdMaxCluster && ctas * kVdWarps * 32 * kVdAhead < vocab) ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, seqs);
    cfg.blockDim = dim3(kVdWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (ctas > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = ctas;
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
    ZL_CHECK_CUDA(cudaLaunchKernelEx(&cfg, k_verify_drafts, p));
    return ZL_OK;
}
