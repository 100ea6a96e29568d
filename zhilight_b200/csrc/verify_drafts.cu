// Verification of drafted tokens against the target's probabilities from given random numbers (the rejection scheme published as speculative
// sampling by Leviathan et al. and Chen et al., 2023): draft i with word x is taken while u_i q_i(x) < p_i(x).  At the first one refused the word comes
// from the weights max(p - q, 0) of that row, behind the last draft from p itself: the first index whose running sum passes u * (sum of all).
//
// Only that one row of p and q is read whole.  The CTAs of a cluster share the vocabulary, a warp has a run of neighbouring words: a pass for the sums
// of the warps, which every CTA gets from the others' shared memory, then the one warp whose run holds the word goes over its run once more.
// Differences, products and sums are in 64 bits: products of two 32-bit numbers are exact there, sums of probabilities above 2^-29 too, and
// a tie falls as the formula says.  Bound by bytes, the latency of a chain of three loads and a cluster's barrier where there are few sequences.
#include "paged.cuh"
#include "tc2_common.cuh"

namespace zl {

constexpr int kVdWarps = 16, kVdMaxCluster = 8, kVdAhead = 8;

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
    __shared__ int s_taken;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.y, ctas = gridDim.x, cta = blockIdx.x;
    if (ctas > 1) cluster_arrive();   // every CTA runs before another one stores into it
    pdl_trigger();
    pdl_wait();
    const int n = p.count ? min(max(p.count[b], 0), p.k) : p.k;
    if (warp == 0) {
        int taken = 0;
        for (int i0 = 0; i0 < n; i0 += 32) {
            const int i = i0 + lane;
            bool ok = false;
            if (i < n) {
                const int x = p.drafted[(size_t)b * p.k + i];
                if ((unsigned)x < (unsigned)p.vocab) {
                    const double q = p.draft ? (double)p.draft[b * p.d_seq + i * p.d_row + x] : 1.0;
                    ok = (double)p.accept[(size_t)b * p.k + i] * q < (double)p.target[b * p.t_seq + i * p.t_row + x];
                }
            }
            const unsigned m = __ballot_sync(0xffffffffu, ok);
            if (m != 0xffffffffu) {
                taken += __ffs(~m) - 1;
                break;
            }
            taken += 32;
        }
        if (lane == 0) s_taken = min(taken, n);
    }
    __syncthreads();
    const int taken = s_taken;
    const bool refused = taken < n;
    const float* tr = p.target + b * p.t_seq + taken * p.t_row;
    const float* dr = refused && p.draft ? p.draft + b * p.d_seq + taken * p.d_row : nullptr;
    const int skip = refused && !p.draft ? p.drafted[(size_t)b * p.k + taken] : -1;   // a draft without probabilities has all of its own on one word
    // this warp's run
    const int run = cdiv(p.vocab, ctas * kVdWarps), lo = min((cta * kVdWarps + warp) * run, p.vocab), hi = min(lo + run, p.vocab);
    double total = 0.0, before = 0.0, mine = 0.0;
    bool plain = !refused;
    if (ctas > 1) cluster_wait();
    // the weight of a word; what is not finite or not positive counts as none
    auto weigh = [&](float a, float q, int i) {
        const double w = plain ? (double)a : (i == skip ? (double)a - 1.0 : (double)a - (double)q);
        return w > 0.0 && w < INFINITY ? w : 0.0;
    };
    for (;;) {
        const float* d2 = plain ? nullptr : dr;
        double s[2] = {0.0, 0.0};
        for (int i = lo + lane; i < hi; i += 32 * kVdAhead) {
            float a[kVdAhead], q[kVdAhead];
#pragma unroll
            for (int u = 0; u < kVdAhead; ++u) {
                const int at = i + 32 * u;
                a[u] = at < hi ? tr[at] : 0.f;
                q[u] = d2 && at < hi ? d2[at] : 0.f;
            }
#pragma unroll
            for (int u = 0; u < kVdAhead; ++u) s[u & 1] += weigh(a[u], q[u], i + 32 * u);
        }
        mine = s[0] + s[1];
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
        total = before = 0.0;
        for (int c = 0; c < ctas; ++c)
            for (int w = 0; w < kVdWarps; ++w) {
                if (c == cta && w == warp) before = total;
                total += part[c][w];
            }
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
    int owner = -1, last = -1;
    {
        double sum = 0.0;
        for (int c = 0; c < ctas; ++c)
            for (int w = 0; w < kVdWarps; ++w) {
                if (part[c][w] > 0.0) last = c * kVdWarps + w;
                sum += part[c][w];
                if (owner < 0 && sum > goal) owner = c * kVdWarps + w;
            }
    }
    if (owner < 0) owner = last;
    if (owner != cta * kVdWarps + warp) return;
    double run_sum = before;
    int word = -1;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        const double w = i < hi ? weigh(tr[i], plain || !dr ? 0.f : dr[i], i) : 0.0;
        double up = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += v;
        }
        const unsigned some = __ballot_sync(0xffffffffu, w > 0.0), past = __ballot_sync(0xffffffffu, w > 0.0 && run_sum + up > goal);
        if (past) {
            word = i0 + __ffs(past) - 1;
            break;
        }
        if (some) word = i0 + 31 - __clz(some);
        run_sum += __shfl_sync(0xffffffffu, up, 31);
    }
    if (lane == 0) p.tokens[(size_t)b * (p.k + 1) + taken] = word;
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
