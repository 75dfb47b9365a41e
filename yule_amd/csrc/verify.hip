// verify.hip — verification of drafted tokens (yule_hip_verify_drafts).
//
// Draft i of a sequence is kept while u_i q_i(x_i) < p_i(x_i): with u uniform in
// [0, 1) that happens with probability min(1, p / q).  At the first draft a that
// is not kept the answer goes on with a token of weights max(p_a - q_a, 0), else
// (all kept) of weights p_a, picked where the running sum passes u_n times the
// whole: together the tokens are distributed as the target's own.  Products of
// two f32 are exact in f64, and sums are f64: a vocabulary's weights in f32 would
// move the pick by up to 2^-24 x its size.
//
// One row of p and one of q is all that has to be read (the drafts' own
// probabilities besides): bandwidth for a batch, latency for a single request.
// The rows are cut into chunks of 4096 values, one workgroup each, which leave
// their sums; a second launch finds the chunk that the pick falls into and walks
// that one again.
#include <cmath>

#include "batch_plan.h"
#include "internal.h"

namespace yule {

struct VerifyArgs {
    const float *p, *q;
    uint64_t ps, qs;             // elements between rows
    const uint32_t *drafts;      // [n_seqs][n_draft]
    const float *u;              // [n_seqs][n_draft + 1]
    const uint32_t *lens;        // drafts of each sequence, or null
    uint32_t *accepted, *tokens; // [n_seqs], [n_seqs][n_draft + 1]
    uint32_t n_draft, vocab, chunks;
    VerifySum *sums;             // [n_seqs][chunks]
};

// a weight: what is not a positive number counts as nothing
__device__ __forceinline__ double weight(double x) { return x > 0.0 ? x : 0.0; }

// kept drafts of sequence s (the same in every lane of every wave that asks)
__device__ __forceinline__ uint32_t kept(const VerifyArgs &a, uint32_t s, uint32_t lane, uint32_t *count) {
    uint32_t n = a.lens ? a.lens[s] : a.n_draft;
    n = n < a.n_draft ? n : a.n_draft;
    *count = n;
    for (uint32_t i0 = 0; i0 < n; i0 += 64) {
        const uint32_t i = i0 + lane;
        bool stop = i >= n;
        if (!stop) {
            const uint32_t x = a.drafts[(size_t)s * a.n_draft + i];
            if (x < a.vocab) {
                const double u = a.u[(size_t)s * (a.n_draft + 1) + i];
                const double q = a.q[((size_t)s * a.n_draft + i) * a.qs + x];
                stop = !(u * q < (double)a.p[((size_t)s * (a.n_draft + 1) + i) * a.ps + x]);
            } else {
                stop = true;   // not a token: no probability
            }
        }
        const uint64_t stops = __ballot(stop);
        if (stops) return i0 + (uint32_t)__builtin_ctzll(stops);
    }
    return n;
}

// the rows that the next token of sequence s comes from (q null: all kept)
__device__ __forceinline__ void rows_of(const VerifyArgs &a, uint32_t s, uint32_t kept, uint32_t count, const float **p,
                                        const float **q) {
    *p = a.p + ((size_t)s * (a.n_draft + 1) + kept) * a.ps;
    *q = kept < count ? a.q + ((size_t)s * a.n_draft + kept) * a.qs : nullptr;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int d = 32; d; d /= 2) x += __shfl_xor(x, d, 64);
    return x;
}
__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
    for (int d = 32; d; d /= 2) {
        const int y = __shfl_xor(x, d, 64);
        x = x > y ? x : y;
    }
    return x;
}

__global__ __launch_bounds__(256) void verify_sums_kernel(VerifyArgs a) {
    __shared__ double sr[4], sp[4];
    __shared__ int lr[4], lp[4];
    const uint32_t s = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, tid = threadIdx.x, lane = tid & 63u;
    uint32_t count;
    const uint32_t n = kept(a, s, lane, &count);
    const float *p, *q;
    rows_of(a, s, n, count, &p, &q);
    const uint32_t x0 = chunk * kVerifyChunk, x1 = a.vocab - x0 < kVerifyChunk ? a.vocab : x0 + kVerifyChunk;
    double rest = 0.0, whole = 0.0;   // of max(p - q, 0), of p
    int last_rest = -1, last_whole = -1;
    for (uint32_t x = x0 + tid; x < x1; x += 256) {
        const double pv = p[x], w = weight(pv), r = q ? weight(pv - (double)q[x]) : w;
        rest += r;
        whole += w;
        if (r > 0.0) last_rest = (int)x;
        if (w > 0.0) last_whole = (int)x;
    }
    rest = wave_sum(rest);
    whole = wave_sum(whole);
    last_rest = wave_max(last_rest);
    last_whole = wave_max(last_whole);
    if (lane == 0) {
        sr[tid >> 6] = rest, sp[tid >> 6] = whole;
        lr[tid >> 6] = last_rest, lp[tid >> 6] = last_whole;
    }
    __syncthreads();
    if (tid == 0) {
        VerifySum v = {sr[0], sp[0], lr[0], lp[0]};
        for (int i = 1; i < 4; i++) {
            v.rest += sr[i];
            v.whole += sp[i];
            v.last_rest = lr[i] > v.last_rest ? lr[i] : v.last_rest;
            v.last_whole = lp[i] > v.last_whole ? lp[i] : v.last_whole;
        }
        a.sums[blockIdx.x] = v;
    }
}

// a workgroup per sequence
__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyArgs a) {
    __shared__ double part[256];
    __shared__ uint32_t found;
    const uint32_t s = blockIdx.x, tid = threadIdx.x, lane = tid & 63u;
    uint32_t count;
    const uint32_t n = kept(a, s, lane, &count);
    const float *p, *q;
    rows_of(a, s, n, count, &p, &q);
    const VerifySum *sums = a.sums + (size_t)s * a.chunks;
    // every thread walks the chunks in order: the same additions everywhere
    double rest = 0.0, whole = 0.0;
    for (uint32_t c = 0; c < a.chunks; c++) {
        rest += sums[c].rest;
        whole += sums[c].whole;
    }
    const bool of_rest = rest > 0.0;   // (rounding may leave p = q at a draft that is not kept: then p itself)
    const double target = (double)a.u[(size_t)s * (a.n_draft + 1) + a.n_draft] * (of_rest ? rest : whole);
    double sum = 0.0;
    uint32_t at = a.chunks;
    int last = -1;
    for (uint32_t c = 0; c < a.chunks; c++) {
        const double w = of_rest ? sums[c].rest : sums[c].whole;
        const int l = of_rest ? sums[c].last_rest : sums[c].last_whole;
        if (l >= 0) last = l;
        if (sum + w > target) {
            at = c;
            break;
        }
        sum += w;
    }
    // (not passed at all: u or a rounding at the very end; the last token that has a weight.  None has: no token)
    uint32_t token = last < 0 ? YULE_NO_TOKEN : (uint32_t)last;
    if (at < a.chunks) {
        const uint32_t x0 = at * kVerifyChunk, x1 = a.vocab - x0 < kVerifyChunk ? a.vocab : x0 + kVerifyChunk;
        constexpr uint32_t EACH = kVerifyChunk / 256;
        auto w_of = [&](uint32_t x) {
            if (x >= x1) return 0.0;
            const double pv = p[x];
            return of_rest && q ? weight(pv - (double)q[x]) : weight(pv);
        };
        double mine = 0.0;
        for (uint32_t i = 0; i < EACH; i++) mine += w_of(x0 + tid * EACH + i);
        part[tid] = mine;
        if (tid == 0) found = token;   // (last weighted token of the chunk, should its sum round below the target)
        __syncthreads();
        for (uint32_t i = 0; i < tid; i++) sum += part[i];
        __syncthreads();
        for (uint32_t i = 0; i < EACH && mine > 0.0; i++) {
            sum += w_of(x0 + tid * EACH + i);
            if (sum > target) {
                atomicMin(&found, x0 + tid * EACH + i);
                break;
            }
        }
        __syncthreads();
        token = found;
    }
    for (uint32_t i = tid; i <= a.n_draft; i += 256)
        a.tokens[(size_t)s * (a.n_draft + 1) + i] = i < n    ? a.drafts[(size_t)s * a.n_draft + i]
                                                    : i == n ? token
                                                             : YULE_NO_TOKEN;
    if (tid == 0) a.accepted[s] = n;
}

}  // namespace yule

using namespace yule;

extern "C" int yule_hip_verify_drafts(yule_hip_backend *be, const yule_rows *target, const yule_rows *draft,
                                      yule_buffer draft_tokens, yule_buffer uniforms, yule_buffer draft_lens,
                                      yule_buffer accepted, yule_buffer tokens, uint32_t n_seqs, uint32_t n_draft,
                                      uint32_t vocab) {
    return guarded("verify_drafts", be, [&]() -> int {
        if (!vocab || vocab > kMaxVocab) return set_error(YULE_ERR_INVALID, "verify_drafts: vocab must be 1..2^30");
        if (n_draft > kMaxDrafts) return set_error(YULE_ERR_INVALID, "verify_drafts: more than 1024 drafts");
        const uint64_t rows_p = (uint64_t)n_seqs * (n_draft + 1), rows_q = (uint64_t)n_seqs * n_draft;
        VerifyArgs a = {};
        void *pp, *pq = nullptr, *pd = nullptr, *pu, *pl = nullptr, *pa, *pt;
        int rc;
        if ((rc = rows_ptr(be, target, rows_p, vocab, 4, 4, "verify_drafts (target)", &pp)) ||
            (n_draft && (rc = rows_ptr(be, draft, rows_q, vocab, 4, 4, "verify_drafts (draft)", &pq))) ||
            (n_draft && (rc = get_buffer(be, draft_tokens, rows_q * 4, &pd, "verify_drafts (draft_tokens)"))) ||
            (rc = get_buffer(be, uniforms, rows_p * 4, &pu, "verify_drafts (uniforms)")) ||
            (draft_lens && (rc = get_buffer(be, draft_lens, (size_t)n_seqs * 4, &pl, "verify_drafts (draft_lens)"))) ||
            (rc = get_buffer(be, accepted, (size_t)n_seqs * 4, &pa, "verify_drafts (accepted)")) ||
            (rc = get_buffer(be, tokens, rows_p * 4, &pt, "verify_drafts (tokens)")))
            return rc;
        const yule_buffer in[] = {target->buffer, n_draft ? draft->buffer : 0, n_draft ? draft_tokens : 0, uniforms, draft_lens};
        for (yule_buffer b : in)
            if (b == accepted || b == tokens) return set_error(YULE_ERR_INVALID, "verify_drafts: an input and an output alias");
        if (accepted == tokens) return set_error(YULE_ERR_INVALID, "verify_drafts: outputs alias");
        if (!n_seqs) return YULE_OK;
        const uint64_t chunks = (vocab + kVerifyChunk - 1) / kVerifyChunk;
        if (n_seqs * chunks > kMaxWorkgroups) return set_error(YULE_ERR_INVALID, "verify_drafts: too many rows for one call");
        ScratchLease ws;   // held until both launches are enqueued
        if ((rc = get_scratch(be, n_seqs * chunks * sizeof(VerifySum), &ws))) return rc;
        a.p = static_cast<const float *>(pp), a.q = static_cast<const float *>(pq);
        a.ps = target->stride, a.qs = n_draft ? draft->stride : 0;
        a.drafts = static_cast<const uint32_t *>(pd), a.u = static_cast<const float *>(pu);
        a.lens = static_cast<const uint32_t *>(pl);
        a.accepted = static_cast<uint32_t *>(pa), a.tokens = static_cast<uint32_t *>(pt);
        a.n_draft = n_draft, a.vocab = vocab, a.chunks = (uint32_t)chunks;
        a.sums = static_cast<VerifySum *>(ws.ptr);
        hipLaunchKernelGGL(verify_sums_kernel, dim3((uint32_t)(n_seqs * chunks)), dim3(256), 0, be->stream, a);
        if ((rc = check_launch("verify_drafts (sums)"))) return rc;
        hipLaunchKernelGGL(verify_pick_kernel, dim3(n_seqs), dim3(256), 0, be->stream, a);
        return check_launch("verify_drafts (pick)");
    });
}
