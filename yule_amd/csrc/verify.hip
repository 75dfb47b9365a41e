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
// One launch: the rows are cut into chunks of 4096 values, a workgroup each, which
// leave their sums; the one that takes a sequence's last ticket finds the chunk that
// the pick falls into and loads that one again.  (A workgroup of 1024 threads for a
// whole row of 32000 values needs no tickets, but is no faster up to 64 sequences:
// 7.4 against 7.0 us for one, 10.4 against 10.6 for 64; 200: 12.1 against 16.2.)
// A row of one chunk takes 4.9 us; a ticket, the sums and the chunk once more add
// 2, and 64 requests of 32000 values, 16 MB, 10.6 in all.
#include <type_traits>

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
    uint32_t n_draft, vocab, chunks, seq0;
    double *sums;                // [sequences of the launch][chunks]
    uint32_t *tickets;           // one of kVerifyTicketWords for each sequence of the launch, zero before and after
};

// a weight: what is not a positive number counts as nothing
__device__ __forceinline__ double weight(double x) { return x > 0.0 ? x : 0.0; }

// kept drafts of sequence s (the same in every lane of every wave that asks)
__device__ __forceinline__ uint32_t kept(const VerifyArgs &a, uint32_t s, uint32_t lane, uint32_t *count) {
    // (what does not depend on another load is loaded first)
    uint32_t n = a.lens ? a.lens[s] : a.n_draft;
    *count = 0;
    if (!a.n_draft) return 0;
    for (uint32_t i0 = 0; i0 < a.n_draft; i0 += 64) {
        const uint32_t i = i0 + lane < a.n_draft ? i0 + lane : a.n_draft - 1u;
        const uint32_t x = a.drafts[(size_t)s * a.n_draft + i], xc = x < a.vocab ? x : 0u;
        const double u = a.u[(size_t)s * (a.n_draft + 1) + i];
        const double q = a.q[((size_t)s * a.n_draft + i) * a.qs + xc];
        const double p = a.p[((size_t)s * (a.n_draft + 1) + i) * a.ps + xc];
        n = n < a.n_draft ? n : a.n_draft;
        *count = n;
        // (x of vocab or more is no token and has no probability)
        const uint64_t stops = __ballot(i0 + lane >= n || x >= a.vocab || !(u * q < p));
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

// inclusive sums over the wave's lanes, by DPP row shifts and row broadcasts
__device__ __forceinline__ double wave_scan(double x) {
    auto step = [&](auto ctrl, auto rows) {   // lanes without a source add 0
        constexpr int CTRL = decltype(ctrl)::value, ROWS = decltype(rows)::value;
        const uint64_t b = __builtin_bit_cast(uint64_t, x);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
        x += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});   // row_shr 1, 2, 4, 8
    step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});   // row_bcast 15, 31
    step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
    return x;
}
__device__ __forceinline__ double lane_of(double x, uint32_t l) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), (int)l) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, (int)l));
}

// values x .. x + 3 of a row of n, 0 past its end: one load where the row allows it
__device__ __forceinline__ void load4(const float *row, uint32_t x, uint32_t n, bool aligned, float v[4]) {
    if (aligned && x + 4 <= n) {
        const float4 f = *reinterpret_cast<const float4 *>(row + x);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) v[e] = x + e < n ? row[x + e] : 0.f;
    }
}

// A thread has 4 J values of a chunk, 4 NT j + 4 tid .., so a wave's are 256 in a row
// (a group), NG groups a chunk.  Sums are taken in one order, whoever takes the
// last ticket.
__global__ __launch_bounds__(256) void verify_kernel(VerifyArgs a) {
    constexpr uint32_t NT = 256, J = 4, NW = NT / 64, NG = NW * J, CHUNK = kVerifyChunk;
    static_assert(CHUNK == 4 * NT * J && NG <= 64);
    __shared__ double part[NG];   // the groups' sums
    __shared__ uint32_t shared_last, token;
    const uint32_t s = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, seq = a.seq0 + s;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    uint32_t count;
    const uint32_t n = kept(a, seq, lane, &count);
    const float *p, *q;
    rows_of(a, seq, n, count, &p, &q);

    float pv[J][4], qv[J][4];   // this thread's values of a chunk
    auto four = [&](uint32_t j, double w[4]) {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) w[e] = weight(q ? (double)pv[j][e] - (double)qv[j][e] : (double)pv[j][e]);
        return (w[0] + w[1]) + (w[2] + w[3]);
    };
    double group, upto;         // lane's group (of the first NG lanes), and the sum up to and with it
    auto weigh = [&](uint32_t c) {   // the chunk's sum (in every lane)
        const bool p_al = (reinterpret_cast<uintptr_t>(p) & 15u) == 0, q_al = (reinterpret_cast<uintptr_t>(q) & 15u) == 0;
#pragma unroll
        for (uint32_t j = 0; j < J; j++) load4(p, c * CHUNK + 4 * NT * j + 4 * tid, a.vocab, p_al, pv[j]);
        if (q) {
#pragma unroll
            for (uint32_t j = 0; j < J; j++) load4(q, c * CHUNK + 4 * NT * j + 4 * tid, a.vocab, q_al, qv[j]);
        }
#pragma unroll
        for (uint32_t j = 0; j < J; j++) {
            double w[4];
            const double sum = wave_scan(four(j, w));
            if (lane == 63) part[NW * j + wave] = sum;
        }
        __syncthreads();
        group = lane < NG ? part[lane] : 0.0;
        upto = wave_scan(group);
        return lane_of(upto, 63);
    };
    auto put = [&](uint32_t c, double sum) {   // (one lane) complete at device scope when it returns, without a cache-wide fence
        __hip_atomic_store(reinterpret_cast<uint64_t *>(a.sums + (size_t)s * a.chunks + c), __builtin_bit_cast(uint64_t, sum),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
    };

    double all = weigh(chunk), before = 0.0;
    uint32_t at = 0;
    if (a.chunks > 1) {
        if (tid == 0) {
            put(chunk, all);
            uint32_t *ticket = a.tickets + kVerifyTicketWords * s;
            const bool mine = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.chunks - 1u;
            if (mine) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            shared_last = mine;
        }
        __syncthreads();
        if (!shared_last) return;
    }
    const double u = a.u[(size_t)seq * (a.n_draft + 1) + a.n_draft];
    double target;
    for (;;) {   // (twice if max(p - q, 0) is zero everywhere)
        if (a.chunks > 1) {   // every wave for itself: all the sums, then the chunk that the target falls into
            double sum = 0.0;
            auto sum_of = [&](uint32_t c) {
                return c < a.chunks ? __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<uint64_t *>(a.sums + (size_t)s * a.chunks + c),
                                                                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
                                    : 0.0;
            };
            const double first = sum_of(lane);
            all = lane_of(wave_scan(first), 63);
            for (uint32_t c0 = 64; c0 < a.chunks; c0 += 64) all += lane_of(wave_scan(sum_of(c0 + lane)), 63);
            target = u * all;
            at = 0;
            for (uint32_t c0 = 0; c0 < a.chunks; c0 += 64) {
                const double mine = c0 ? sum_of(c0 + lane) : first, up = wave_scan(mine);
                const uint64_t some = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && sum + up > target);
                if (some) {   // the first past it, or so far the last that has a weight (u, or a rounding, at the very end)
                    const uint32_t l = past ? (uint32_t)__builtin_ctzll(past) : 63u - (uint32_t)__builtin_clzll(some);
                    at = c0 + l;
                    before = l ? sum + lane_of(up, l - 1u) : sum;
                }
                if (past) break;
                sum += lane_of(up, 63);
            }
        } else {
            target = u * all;
        }
        if (all > 0.0 || !q) break;
        // p = q at a draft that is not kept (roundings can leave that, or a draft that is no token): p itself
        q = nullptr;
        __syncthreads();   // (part has been read)
        for (uint32_t c = 0; c < a.chunks; c++) {
            all = weigh(c);
            if (tid == 0 && a.chunks > 1) put(c, all);
            __syncthreads();
        }
    }
    if (a.chunks > 1) {
        __syncthreads();
        (void)weigh(at);
    }
    // The group, then the four, then the value: the first that passes the target, or (sums taken in other orders may
    // round to either side of it) the last that has a weight.
    if (tid == 0) token = YULE_NO_TOKEN;   // nothing has a weight
    {
        const uint64_t some = __ballot(group > 0.0), past = __ballot(group > 0.0 && before + upto > target);
        const uint32_t i = past ? (uint32_t)__builtin_ctzll(past) : some ? 63u - (uint32_t)__builtin_clzll(some) : 0u;
        const double sum = i ? before + lane_of(upto, i - 1u) : before;
        __syncthreads();
        if (some && wave == i % NW) {
            double w[4] = {0.0, 0.0, 0.0, 0.0}, here = 0.0;
#pragma unroll
            for (uint32_t j = 0; j < J; j++)
                if (j == i / NW) here = four(j, w);
            const double up = sum + wave_scan(here);
            const uint64_t any = __ballot(here > 0.0), over = __ballot(here > 0.0 && up > target);
            const uint32_t m = over ? (uint32_t)__builtin_ctzll(over) : any ? 63u - (uint32_t)__builtin_clzll(any) : 0u;
            double r = m ? lane_of(up, m - 1u) : sum;
            if (lane == m && any) {
                uint32_t pick = 0;
                bool got = false;
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    r += w[e];
                    if (w[e] > 0.0 && !got) pick = e;
                    got = got || (w[e] > 0.0 && r > target);
                }
                token = at * CHUNK + 4 * NT * (i / NW) + 4 * tid + pick;
            }
        }
    }
    __syncthreads();
    for (uint32_t i = tid; i <= a.n_draft; i += NT)
        a.tokens[(size_t)seq * (a.n_draft + 1) + i] = i < n    ? a.drafts[(size_t)seq * a.n_draft + i]
                                                      : i == n ? token
                                                               : YULE_NO_TOKEN;
    if (tid == 0) a.accepted[seq] = n;
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
        if ((rc = rows_ptr(be, target, rows_p, vocab, 4, 4, kAnyStride, "verify_drafts (target)", &pp)) ||
            (n_draft && (rc = rows_ptr(be, draft, rows_q, vocab, 4, 4, kAnyStride, "verify_drafts (draft)", &pq))) ||
            (n_draft && (rc = get_buffer(be, draft_tokens, rows_q * 4, &pd, "verify_drafts (draft_tokens)", 0, true))) ||
            (rc = get_buffer(be, uniforms, rows_p * 4, &pu, "verify_drafts (uniforms)", 0, true)) ||
            (draft_lens && (rc = get_buffer(be, draft_lens, (size_t)n_seqs * 4, &pl, "verify_drafts (draft_lens)", 0, true))) ||
            (rc = get_buffer(be, accepted, (size_t)n_seqs * 4, &pa, "verify_drafts (accepted)", 0, true)) ||
            (rc = get_buffer(be, tokens, rows_p * 4, &pt, "verify_drafts (tokens)", 0, true)))
            return rc;
        const yule_buffer in[] = {target->buffer, n_draft ? draft->buffer : 0, n_draft ? draft_tokens : 0, uniforms, draft_lens};
        for (yule_buffer b : in)
            if (b == accepted || b == tokens) return set_error(YULE_ERR_INVALID, "verify_drafts: an input and an output alias");
        if (accepted == tokens) return set_error(YULE_ERR_INVALID, "verify_drafts: outputs alias");
        if (!n_seqs) return YULE_OK;
        const uint64_t chunks = (vocab + kVerifyChunk - 1) / kVerifyChunk;
        if ((uint64_t)n_seqs * chunks > kMaxWorkgroups) return set_error(YULE_ERR_INVALID, "verify_drafts: too many rows for one call");
        ScratchLease ws;   // held until the launches are enqueued
        if ((rc = get_scratch(be, (n_seqs < kVerifyTickets ? n_seqs : kVerifyTickets) * chunks * sizeof(double), &ws))) return rc;
        a.p = static_cast<const float *>(pp), a.q = static_cast<const float *>(pq);
        a.ps = target->stride, a.qs = n_draft ? draft->stride : 0;
        a.drafts = static_cast<const uint32_t *>(pd), a.u = static_cast<const float *>(pu);
        a.lens = static_cast<const uint32_t *>(pl);
        a.accepted = static_cast<uint32_t *>(pa), a.tokens = static_cast<uint32_t *>(pt);
        a.n_draft = n_draft, a.vocab = vocab, a.chunks = (uint32_t)chunks;
        a.sums = static_cast<double *>(ws.ptr);
        a.tickets = static_cast<uint32_t *>(be->verify_ws);
        for (uint32_t s0 = 0; s0 < n_seqs; s0 += kVerifyTickets) {   // (a ticket each)
            const uint32_t now = n_seqs - s0 < kVerifyTickets ? n_seqs - s0 : kVerifyTickets;
            a.seq0 = s0;
            hipLaunchKernelGGL(verify_kernel, dim3((uint32_t)(now * chunks)), dim3(256), 0, be->stream, a);
            if ((rc = check_launch("verify_drafts"))) return rc;
        }
        return YULE_OK;
    });
}
