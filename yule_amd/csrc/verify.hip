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
// One launch: the rows are cut into chunks of 4096 values, a workgroup each,
// which leave their sums; the workgroup that takes a sequence's last ticket finds
// the chunk that the pick falls into and walks that one again.
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
    VerifySum *sums;             // [sequences of the launch][chunks]
    uint32_t *tickets;           // [sequences of the launch], zero before and after
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
__device__ __forceinline__ double last_lane(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), 63) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63));
}
__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
    for (int d = 32; d; d /= 2) {
        const int y = __shfl_xor(x, d, 64);
        x = x > y ? x : y;
    }
    return x;
}

// Values x0 + 1024 j + 4 tid + e (j, e < 4) of a row in this thread's registers,
// 0 past n: 16-byte loads where the row allows them.
__device__ __forceinline__ void load_chunk(const float *row, uint32_t x0, uint32_t n, uint32_t tid, float v[4][4]) {
    const bool whole = x0 + kVerifyChunk <= n && (reinterpret_cast<uintptr_t>(row) & 15u) == 0;
    if (whole) {
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const float4 f = *reinterpret_cast<const float4 *>(row + x0 + 1024 * j + 4 * tid);
            v[j][0] = f.x, v[j][1] = f.y, v[j][2] = f.z, v[j][3] = f.w;
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint32_t x = x0 + 1024 * j + 4 * tid + e;
                const float f = row[x < n ? x : n - 1u];
                v[j][e] = x < n ? f : 0.f;
            }
    }
}

// A workgroup per chunk; the one that takes its sequence's last ticket picks and
// answers.  Sums are taken in one order, whoever is last.
__global__ __launch_bounds__(256) void verify_kernel(VerifyArgs a) {
    __shared__ double part[16];   // sums of 256 weights each: 1024 j + 256 wave ..
    __shared__ int lasts[4];      // last places that have a weight, by wave
    __shared__ double target, before;
    __shared__ uint32_t is_last, at, token, again;
    const uint32_t s = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, seq = a.seq0 + s;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    uint32_t count;
    const uint32_t n = kept(a, seq, lane, &count);
    const float *p, *q;
    rows_of(a, seq, n, count, &p, &q);

    double w[4][4];   // this thread's weights of a chunk
    auto weigh = [&](uint32_t c) {
        float pv[4][4], qv[4][4];
        load_chunk(p, c * kVerifyChunk, a.vocab, tid, pv);
        if (q) load_chunk(q, c * kVerifyChunk, a.vocab, tid, qv);
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) w[j][e] = weight(q ? (double)pv[j][e] - (double)qv[j][e] : (double)pv[j][e]);
            const double sum = last_lane(wave_scan((w[j][0] + w[j][1]) + (w[j][2] + w[j][3])));
            if (lane == 0) part[4 * j + wave] = sum;
        }
        int last = -1;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
#pragma unroll
            for (uint32_t e = 0; e < 4; e++)
                if (w[j][e] > 0.0) last = (int)(c * kVerifyChunk + 1024 * j + 4 * tid + e);
        last = wave_max(last);
        if (lane == 0) lasts[wave] = last;
        __syncthreads();
    };
    // (every thread) the chunk that was weighed
    auto chunk_sum = [&](int *last) {
        double sum = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) sum += part[i];
        *last = -1;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) *last = lasts[i] > *last ? lasts[i] : *last;
        return sum;
    };
    auto put = [&](uint32_t c, double sum, int last) {   // (one lane)
        uint64_t *o = reinterpret_cast<uint64_t *>(a.sums + (size_t)s * a.chunks + c);
        __hip_atomic_store(o, __builtin_bit_cast(uint64_t, sum), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(o + 1, (uint64_t)(int64_t)last, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };

    weigh(chunk);
    if (wave == 0) {
        uint32_t mine = 1;
        int last;
        const double sum = chunk_sum(&last);
        if (a.chunks > 1) {
            if (lane == 0) {
                // complete at device scope before the ticket is taken (no cache-wide fence)
                put(chunk, sum, last);
                __atomic_signal_fence(__ATOMIC_SEQ_CST);
                __builtin_amdgcn_s_waitcnt(0);
                __atomic_signal_fence(__ATOMIC_SEQ_CST);
                mine = __hip_atomic_fetch_add(a.tickets + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.chunks - 1u;
                if (mine) __hip_atomic_store(a.tickets + s, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            mine = __builtin_amdgcn_readfirstlane(mine);
        }
        if (lane == 0) is_last = mine;
    }
    __syncthreads();
    if (!is_last) return;

    for (;;) {
        // the chunk that the pick falls into, 64 chunks at a time
        if (wave == 0) {
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
            double c_sum;   // lane's chunk (without others this one)
            int c_last;
            auto load_sums = [&](uint32_t c) {
                int last;
                const double sum = chunk_sum(&last);
                c_sum = c == 0 ? sum : 0.0;
                c_last = c == 0 ? last : -1;
                if (a.chunks > 1) {
                    c_sum = 0.0, c_last = -1;
                    if (c < a.chunks) {
                        const uint64_t *o = reinterpret_cast<const uint64_t *>(a.sums + (size_t)s * a.chunks + c);
                        c_sum = __builtin_bit_cast(double, __hip_atomic_load(o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
                        c_last = (int)__hip_atomic_load(o + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
                }
            };
            double all = 0.0;
            int last = -1;
            for (uint32_t c0 = 0; c0 < a.chunks; c0 += 64) {
                load_sums(c0 + lane);
                all += last_lane(wave_scan(c_sum));
                const int l = wave_max(c_last);
                last = l > last ? l : last;
            }
            const double t = (double)a.u[(size_t)seq * (a.n_draft + 1) + a.n_draft] * all;
            double sum = 0.0;
            uint32_t hit = a.chunks;
            for (uint32_t c0 = 0; c0 < a.chunks; c0 += 64) {
                if (a.chunks > 64) load_sums(c0 + lane);
                const double upto = wave_scan(c_sum);
                const uint64_t past = __ballot(c0 + lane < a.chunks && sum + upto > t);
                if (past) {
                    const int l = __builtin_ctzll(past);
                    hit = c0 + (uint32_t)l;
                    const double up = __shfl(upto, l ? l - 1 : 0, 64);
                    if (l) sum += up;
                    break;
                }
                sum += last_lane(upto);
            }
            if (lane == 0) {
                // not passed at all (u, or a rounding, at the very end): the last token that has a weight, if one has
                token = last < 0 ? YULE_NO_TOKEN : (uint32_t)last;
                target = t, before = sum, at = hit;
                again = last < 0 && q;
            }
        }
        __syncthreads();
        if (!again) break;
        // p = q at a draft that is not kept (roundings can leave that, or a draft that is no token): p itself
        q = nullptr;
        for (uint32_t c = 0; c < a.chunks; c++) {
            weigh(c);
            if (tid == 0 && a.chunks > 1) {
                int last;
                const double sum = chunk_sum(&last);
                put(c, sum, last);
            }
            if (c + 1 < a.chunks) __syncthreads();
        }
        if (tid == 0) {   // (read by the first wave only, which waits for them here)
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
            __builtin_amdgcn_s_waitcnt(0);
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
        }
        __syncthreads();
    }
    if (at < a.chunks) {
        if (a.chunks > 1) weigh(at);   // (one chunk: still there)
        // The 256 values, then the four, then the value.  (Sums taken in other orders may round to either side of the
        // target: then the last with a weight.)
        double run = before, sum = before;
        uint32_t i = 0;
        for (uint32_t k = 0; k < 16; k++) {
            if (part[k] > 0.0) {
                i = k;
                sum = run;
                if (run + part[k] > target) break;
            }
            run += part[k];
        }
        if (wave == (i & 3u)) {
            double mine[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
                if (j == i >> 2) {
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++) mine[e] = w[j][e];
                }
            const double four = (mine[0] + mine[1]) + (mine[2] + mine[3]);
            const double upto = sum + wave_scan(four);
            const uint64_t past = __ballot(upto > target && four > 0.0), some = __ballot(four > 0.0);
            const uint32_t l = past ? (uint32_t)__builtin_ctzll(past) : some ? 63u - (uint32_t)__builtin_clzll(some) : 0u;
            double here = __shfl_up(upto, 1, 64);
            if (lane == 0) here = sum;
            if (lane == l && some) {
                uint32_t pick = 0;
                bool found = false;
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    here += mine[e];
                    if (mine[e] > 0.0 && !found) pick = e;
                    found = found || here > target;
                }
                token = at * kVerifyChunk + 1024 * (i >> 2) + 4 * tid + pick;
            }
        }
    }
    __syncthreads();
    for (uint32_t i = tid; i <= a.n_draft; i += 256)
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
        if ((uint64_t)n_seqs * chunks > kMaxWorkgroups) return set_error(YULE_ERR_INVALID, "verify_drafts: too many rows for one call");
        ScratchLease ws;   // held until the launches are enqueued
        if ((rc = get_scratch(be, (n_seqs < kVerifyTickets ? n_seqs : kVerifyTickets) * chunks * sizeof(VerifySum), &ws))) return rc;
        a.p = static_cast<const float *>(pp), a.q = static_cast<const float *>(pq);
        a.ps = target->stride, a.qs = n_draft ? draft->stride : 0;
        a.drafts = static_cast<const uint32_t *>(pd), a.u = static_cast<const float *>(pu);
        a.lens = static_cast<const uint32_t *>(pl);
        a.accepted = static_cast<uint32_t *>(pa), a.tokens = static_cast<uint32_t *>(pt);
        a.n_draft = n_draft, a.vocab = vocab, a.chunks = (uint32_t)chunks;
        a.sums = static_cast<VerifySum *>(ws.ptr);
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
