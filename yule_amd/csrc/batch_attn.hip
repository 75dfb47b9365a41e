// batch_attn.hip — attention of batches: packed prompts (yule_hip_prompt_attn)
// and new tokens over a shared prefix and their own tails
// (yule_hip_prefix_attn).  Grouped heads, f32, f16 and bf16.
//
// Both are the same walk.  The (query row, query head) pairs of one KV head are
// its "slots", row by row with the group's heads side by side, so a key that is
// read serves every head of the group.  A wave holds 32 slots and walks its keys
// in subtiles of 32 with an online softmax:
//   S^T = K Q^T      keys x slots, a lane holds 16 keys of one slot
//   p = 2^(c S - m), m a running maximum of c S (up to kLag behind, less kRaise), c = log2(e) / sqrt(hd)
//   O^T += V^T P^T   dims x slots; the lane's p are the operand as they lie
// on the 32-row matrix instructions (operand row or column = lane % 32, k from h
// = lane / 32; result column = lane % 32, row = 8 (i / 4) + 4 h + i % 4).  The
// softmax reduces in the lane and across one swap of the halves.  A sum over k
// does not mind the order of k, so 16-byte pieces of K and Q serve as operands
// of any type, and P needs no rearranging: the keys of register i are taken from
// V's rows instead.
#include <cmath>
#include <type_traits>

#include "batch_plan.h"
#include "internal.h"

namespace yule {

typedef int i4v __attribute__((ext_vector_type(4)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t *lds_b;
typedef __attribute__((address_space(3))) s4v *lds_s4;

// ---- matrix instructions by type: 16 bytes of each operand's row per lane
template <typename T>
__device__ __forceinline__ f16v mma16(i4v a, i4v b, f16v c) {
    if constexpr (sizeof(T) == 4) {
        const f4v x = __builtin_bit_cast(f4v, a), y = __builtin_bit_cast(f4v, b);
#pragma unroll
        for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
        return c;
    } else if constexpr (__is_same(T, _Float16)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
    }
}

// Eight weights as an operand, rounded to the type: 2^-8 (bf16) or 2^-11 of each at
// most, as much as the result's own rounding, and of either sign, so that the two
// together stay below 1.5 times the one.  f16 has a fixed step below 2^-14, so that
// many small weights beside a large one would be off together, and lost below 2^-25
// (1700 keys of weight 2^-26: all of them), while the sum has them.  They are taken
// 2^kRaise times as large: off by 2^-32 of the walk's largest weight at most, where
// that is more than 2^-11 of their own.  The weights' sum keeps f32.
template <typename T>
__device__ __forceinline__ i4v pack8(const f16v &s, int at) {
    if constexpr (__is_same(T, _Float16)) {
        h8v r;
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = (_Float16)s[at + j];
        return __builtin_bit_cast(i4v, r);
    } else {
        b8v r;
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = (__bf16)s[at + j];
        return __builtin_bit_cast(i4v, r);
    }
}

// some element of 16 bytes is infinite or NaN
template <typename T>
__device__ __forceinline__ bool not_finite(i4v x) {
    constexpr uint32_t E = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t w = (uint32_t)x[j];
        bad |= (w & E) == E;
        if constexpr (sizeof(T) == 2) bad |= (w & (E << 16)) == (E << 16);
    }
    return bad;
}

// A key that a slot does not see has weight 0, but 0 times an infinity or a NaN
// is not 0: where some slots do not see some keys, V's values that are not finite
// become 0 in LDS (N words of 16 bytes a lane, as the lanes copied them) and are
// added at the end to those that see them.  Their weights do not matter then.
// True (in every lane): there were some.
template <typename T, uint32_t N>
__device__ __forceinline__ bool drop_not_finite(uint8_t *v, uint32_t lane) {
    bool bad = false;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) bad |= not_finite<T>(*reinterpret_cast<const i4v *>(v + 1024 * i + 16 * lane));
    if (!__ballot(bad)) return false;
#pragma unroll 1
    for (uint32_t i = 0; i < N; i++) {
        T *x = reinterpret_cast<T *>(v + 1024 * i + 16 * lane);
#pragma unroll
        for (uint32_t j = 0; j < 16 / sizeof(T); j++) {
            const float f = (float)x[j];
            if (!(__builtin_fabsf(f) < INFINITY)) x[j] = (T)0.f;
        }
    }
    return true;
}
// sums of four dims + the values that are not finite of keys k0 .. k1 - 1 (v: key 0's four)
template <typename T>
__device__ __forceinline__ f4v add_not_finite(f4v o, const uint8_t *v, uint32_t stride, uint32_t k0, uint32_t k1) {
    for (uint32_t k = k0; k < k1; k++) {
        const T *x = reinterpret_cast<const T *>(v + (size_t)k * stride);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float f = (float)x[j];
            if (!(__builtin_fabsf(f) < INFINITY)) o[j] += f;
        }
    }
    return o;
}

// ---- a subtile in LDS: 32 rows of D elements as C 16-byte chunks, chunk c of
// row r at chunk c ^ swizzle(r) of its row.  P rows fill the 256 bytes of all
// banks, and the XOR walks the G chunks that a power of two divides off C: 16
// rows of one chunk (K operands), and 8 rows of two chunks (step 2: V operands),
// lie in different banks.
template <uint32_t C, uint32_t STEP>
__device__ __forceinline__ uint32_t swizzle(uint32_t r) {
    constexpr uint32_t G = C % 16 == 0 ? 16 : C % 8 == 0 ? 8 : C % 4 == 0 ? 4 : 2, P = 16 / G;
    return (STEP * (r / P)) % G;
}

// outside the compiler's memory model, its waits included: every wait for it is
// explicit, and so is the wait state after a scalar write of M0
__device__ __forceinline__ void copy_to_lds(const uint8_t *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base),
                 "s"(__builtin_amdgcn_readfirstlane(lds))
                 : "m0", "memory");
}
template <uint32_t N>
__device__ __forceinline__ void wait_copies() {   // until at most N are in flight
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// x as the compiler knows nothing about it: what is computed from it is computed
// there, and not kept in registers over the loop (operand and copy addresses: a
// few integer operations each, beside hundreds of registers)
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
    asm volatile("; used" : "+v"(x));
    return x;
}

// an address that is the same in every lane, in scalar registers
__device__ __forceinline__ const uint8_t *uniform(uint64_t x) {
    return reinterpret_cast<const uint8_t *>((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 |
                                             (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x));
}

// rows of a cache or activation: address of row 0 of one head, bytes between rows
struct Rows {
    const uint8_t *p;
    uint32_t stride;
};

// the larger of x and the other half's (lane +- 32)
__device__ __forceinline__ float max_halves(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// What weights are taken against: a running maximum m of c S that lags up to kLag
// behind the true one, so that the weight's sum l (this lane's keys) and the sums o
// are rescaled a few times and not with every new maximum of any slot (half of
// the subtiles of a long walk; a sixth of its time), and is kRaise below it.
// Weights reach 2^(kLag + kRaise) then: 2^15 in f16, which ends at 65504.
constexpr float kLag = 8.f;
template <typename T>
constexpr float kRaise = __is_same(T, _Float16) ? 7.f : 0.f;
template <typename T, uint32_t N, uint32_t DT>
__device__ __forceinline__ void new_maximum(const f16v (&s)[N], f16v (&o)[DT], float &m, float &l, float c) {
    float cm = s[0][0];
#pragma unroll
    for (uint32_t n = 0; n < N; n++)
#pragma unroll
        for (int i = n ? 0 : 1; i < 16; i++) cm = fmaxf(cm, s[n][i]);
    cm = max_halves(cm) * c - kRaise<T>;
    if (__ballot(cm > m + kLag)) {
        const float mn = fmaxf(m, cm);
        // (m = -inf: nothing was added yet, and the factor multiplies zeros)
        const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (uint32_t t = 0; t < DT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][i] *= alpha;
    }
}
// scores into weights 2^(c S - m): the product and the difference round once, in the fused multiply-add
template <uint32_t N>
__device__ __forceinline__ void weights(f16v (&s)[N], float m, float &l, float c) {
    const float mb = m == -INFINITY ? 0.f : m;   // nothing seen yet: weights of 0
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            s[n][i] = __builtin_amdgcn_exp2f(fmaf(s[n][i], c, -mb));
            sum[i % 4] += s[n][i];
        }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}
template <typename T, uint32_t N, uint32_t DT>
__device__ __forceinline__ void online_softmax(f16v (&s)[N], f16v (&o)[DT], float &m, float &l, float c) {
    new_maximum<T>(s, o, m, l, c);
    weights(s, m, l, c);
}

// ---- one wave: 32 slots over keys key0, key0 + step, .. < k1 (subtiles of 32)
template <typename T, uint32_t D>
struct WaveAttn {
    static constexpr uint32_t SZ = sizeof(T), RB = D * SZ, C = RB / 16, SUB = 32 * RB;
    static constexpr uint32_t NL = SUB / 1024, NS = RB / 32, DT = D / 32;
    static constexpr uint32_t LDS = 2 * SUB;   // bytes of a wave that walks by itself
    i4v q[NS];    // bytes 32 s + 16 h .. of this lane's slot's query
    f16v o[DT];   // O^T, unnormalised: dim 32 t + 8 (i / 4) + 4 h + i % 4
    float m, l;   // what weights are taken against; this lane's share of their sum

    __device__ __forceinline__ void init(const uint8_t *qrow, uint32_t hb, uint32_t h) {
#pragma unroll
        for (uint32_t s = 0; s < NS; s++) {
            const uint32_t at = 32 * s + 16 * h;
            q[s] = i4v{0, 0, 0, 0};
            if (at < hb) q[s] = *reinterpret_cast<const i4v *>(qrow + at);
        }
#pragma unroll
        for (uint32_t t = 0; t < DT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][i] = 0.f;
        m = -INFINITY;
        l = 0.f;
    }

    // The queries are there: the compiler, which knows nothing of the copies into
    // LDS, would otherwise wait for its loads of them inside the loop, with
    // every copy that is in flight then.
    __device__ __forceinline__ void wait_queries() {
#pragma unroll
        for (uint32_t s = 0; s < NS; s++) asm volatile("; used" : "+v"(q[s]));
    }
    // S^T = K Q^T with K's subtile at k; also(i) after product i
    template <typename F>
    __device__ __forceinline__ f16v scores(const uint8_t *k, uint32_t lane, F also) const {
        const uint32_t r = lane & 31u, h = lane >> 5;
        f16v s;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.f;
#pragma unroll
        for (uint32_t st = 0; st < NS; st++) {
            s = mma16<T>(*reinterpret_cast<const i4v *>(k + r * RB + (((2 * st + h) ^ swizzle<C, 1>(r)) << 4)), q[st], s);
            also(st);
        }
        return s;
    }
    __device__ __forceinline__ f16v scores(const uint8_t *k, uint32_t lane) const { return scores(k, lane, [](uint32_t) {}); }
    // key0: the subtile's first key; the slot sees keys below lim
    __device__ __forceinline__ static void hide(f16v &s, uint32_t key0, uint32_t lim, uint32_t lane) {
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (key0 + 8 * (i / 4) + 4 * (lane >> 5) + i % 4 >= lim) s[i] = -INFINITY;
    }

    // O^T += V^T P^T with V's subtile at v; also(i) after product i
    __device__ __forceinline__ void values(const f16v &s, const uint8_t *v, uint32_t lane) {
        values(s, v, lane, [](uint32_t) {});
    }
    template <typename F>
    __device__ __forceinline__ void values(const f16v &s, const uint8_t *v, uint32_t lane, F also) {
        // the transposing read gives lane l of 16 column l of the four rows that lanes 4 r .. 4 r + 3 point to: here the
        // dims of V^T's rows from four keys
        const uint32_t h = lane >> 5, e = lane & 15u, g = lane >> 4;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const i4v p = pack8<T>(s, 8 * k);
            const uint32_t r0 = 16 * k + 4 * h + (e >> 2), r1 = r0 + 8;
#pragma unroll
            for (uint32_t t = 0; t < DT; t++) {
                const uint32_t ch = 4 * t + 2 * (g & 1u) + ((e & 3u) >> 1), sub = 8 * (e & 1u);
                const s4v a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s4)(lds_b)(v + r0 * RB + ((ch ^ swizzle<C, 2>(r0)) << 4) + sub));
                const s4v a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s4)(lds_b)(v + r1 * RB + ((ch ^ swizzle<C, 2>(r1)) << 4) + sub));
                const auto a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
                o[t] = mma16<T>(__builtin_bit_cast(i4v, a), p, o[t]);
                also(DT * k + t);
            }
        }
    }

    // Keys key, key + step, .. < k1 in subtiles of 32 (lds: this wave's K subtile
    // and V subtile).  A slot sees keys below lim, every slot those below lim_all
    // <= k1.  The next K subtile is on its way while this one's softmax and
    // product with V run, the next V subtile during the next scores: copies
    // complete in order, so "at most NL in flight" says that the older of the
    // two has landed.  True: drop_not_finite dropped something.
    __device__ __forceinline__ bool walk(const Rows &K, const Rows &V, uint32_t hb, uint32_t key, uint32_t step,
                                         uint32_t k1, uint32_t lim, uint32_t lim_all, uint8_t *lds, uint32_t lane,
                                         float c) {
        const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>((lds_b)lds));
        uint8_t *const vt = lds + SUB;
        if (hb < RB) {   // chunks past the head stay zero: copies leave them out
#pragma unroll
            for (uint32_t i = 0; i < 2 * NL; i++) *reinterpret_cast<i4v *>(lds + 1024 * i + 16 * lane) = i4v{0, 0, 0, 0};
            wait_lds();
        }
        using No = std::false_type;
        using Yes = std::true_type;
        // Lane's part of copy i: LDS chunk 64 i + lane of the subtile.  Rows past
        // the last key repeat it (hidden, and the number of copies stays).
        auto copy = [&](const Rows &R, auto is_v, uint32_t at) {
            constexpr uint32_t STEP = decltype(is_v)::value ? 2 : 1;
            const uint8_t *base = uniform(reinterpret_cast<uint64_t>(R.p) + (uint64_t)at * R.stride);
            const uint32_t last = k1 - at - 1u, ln = opaque(lane) & 63u, dst = lds0 + (decltype(is_v)::value ? SUB : 0u);
            auto each = [&](auto whole) {
#pragma unroll
                for (uint32_t i = 0; i < NL; i++) {
                    const uint32_t L = 64 * i + ln, r = L / C, ch = (L % C) ^ swizzle<C, STEP>(r);
                    if (decltype(whole)::value || 16 * ch < hb)
                        copy_to_lds(base, (r < last ? r : last) * R.stride + 16 * ch, dst + 1024 * i);
                }
            };
            if (hb == RB) each(Yes{});
            else each(No{});
        };
        if (key < k1) {
            copy(K, No{}, key);
            copy(V, Yes{}, key);
        }
        wait_queries();
        bool dropped = false;
        auto subtile = [&](auto masked) {
            const bool more = key + step < k1;
            wait_copies<NL>();   // K is there
            f16v s[1] = {scores(lds, opaque(lane) & 63u)};
            wait_lds();
            if (more) copy(K, No{}, key + step);
            if (decltype(masked)::value) hide(s[0], key, lim, lane);
            online_softmax<T>(s, o, m, l, c);
            if (more) wait_copies<NL>();   // V is there
            else wait_copies<0>();
            if (decltype(masked)::value) dropped |= drop_not_finite<T, NL>(vt, lane);
            values(s[0], vt, opaque(lane) & 63u);
            wait_lds();
            if (more) copy(V, Yes{}, key + step);
        };
        for (; key + 32 <= lim_all; key += step) subtile(No{});
        for (; key < k1; key += step) subtile(Yes{});
        return dropped;
    }
};

// ---- the same wave for f32, whose products take four times as long per byte and
// whose rows take twice the LDS: K and V pass through a ring of D / 32 pieces, 32
// keys x 32 dims each, that holds one subtile of either.  Piece j is replaced by
// the piece D / 32 further on as soon as it has been used, so copies are always on
// their way, and half the LDS allows twice the waves: one wave's softmax and waits
// lie under the others' products.
template <uint32_t D>
struct WaveAttn<float, D> {
    static constexpr uint32_t SZ = 4, NS = D / 8, DT = D / 32, C = 8, PIECE = 4096, LDS = DT * PIECE;
    i4v q[NS];    // as above
    f16v o[DT];
    float m, l;

    __device__ __forceinline__ void init(const uint8_t *qrow, uint32_t hb, uint32_t h) {
#pragma unroll
        for (uint32_t s = 0; s < NS; s++) {
            const uint32_t at = 32 * s + 16 * h;
            q[s] = i4v{0, 0, 0, 0};
            if (at < hb) q[s] = *reinterpret_cast<const i4v *>(qrow + at);
        }
#pragma unroll
        for (uint32_t t = 0; t < DT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][i] = 0.f;
        m = -INFINITY;
        l = 0.f;
    }

    __device__ __forceinline__ bool walk(const Rows &K, const Rows &V, uint32_t hb, uint32_t key, uint32_t step,
                                         uint32_t k1, uint32_t lim, uint32_t lim_all, uint8_t *lds, uint32_t lane,
                                         float c) {
        const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>((lds_b)lds));
        if (hb < D * 4) {   // what the copies leave out starts as zeros
#pragma unroll
            for (uint32_t i = 0; i < LDS / 1024; i++) *reinterpret_cast<i4v *>(lds + 1024 * i + 16 * lane) = i4v{0, 0, 0, 0};
            wait_lds();
        }
        // f32 products keep the vector units from anything else (measured: their
        // times add up), so addresses are worked out once: of this lane's part of
        // the four copies of a piece (chunk lane % 8 of row 8 i + lane / 8), and of
        // its operands in a piece (from where the other rows' are constants away).
        uint32_t off[2][4], ka[4], va[2];
        {
            const uint32_t lr = lane >> 3, r = lane & 31u, h = lane >> 5;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                off[0][i] = (8 * i + lr) * K.stride + 16 * ((lane & 7u) ^ swizzle<C, 1>(8 * i + lr));
                off[1][i] = (8 * i + lr) * V.stride + 16 * ((lane & 7u) ^ swizzle<C, 2>(8 * i + lr));
                ka[i] = 128 * r + (((2 * i + h) ^ swizzle<C, 1>(r)) << 4);
            }
            // row 8 (i / 4) + 4 h + i % 4: its swizzle is that of 4 h + i % 4
#pragma unroll
            for (uint32_t i = 0; i < 2; i++)
                va[i] = 128 * 4 * h + (((r >> 2) ^ swizzle<C, 2>(4 * h + 2 * i)) << 4) + 4 * (r & 3u);
        }
        // Piece j of the subtile at key `at`: dims 32 j .. of K, then of V.
        auto copy = [&](uint32_t at, uint32_t j) {
            const bool is_v = j >= DT;
            const Rows &R = is_v ? V : K;
            const uint8_t *base = uniform(reinterpret_cast<uint64_t>(R.p) + (uint64_t)at * R.stride + 128 * (j % DT));
            const uint32_t dst = lds0 + PIECE * (j % DT), left = hb - 128 * (j % DT);   // (hd > D - 32: some of every piece)
            if (k1 - at >= 32 && left >= 128) {
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) copy_to_lds(base, off[is_v][i], dst + 1024 * i);
            } else {   // rows past the last key repeat it (hidden, and the number of copies stays)
                const uint32_t last = k1 - at - 1u, ln = opaque(lane) & 63u;
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    const uint32_t r = 8 * i + (ln >> 3), ch = 16 * ((ln & 7u) ^ (is_v ? swizzle<C, 2>(r) : swizzle<C, 1>(r)));
                    if (ch < left) copy_to_lds(base, (r < last ? r : last) * R.stride + ch, dst + 1024 * i);
                }
            }
        };
        if (key < k1) {
#pragma unroll
            for (uint32_t j = 0; j < DT; j++) copy(key, j);
        }
#pragma unroll
        for (uint32_t s = 0; s < NS; s++) asm volatile("; used" : "+v"(q[s]));   // (as wait_queries)
        bool dropped = false;
        auto subtile = [&](auto masked) {
            const bool more = key + step < k1;
            f16v s[1];
#pragma unroll
            for (int i = 0; i < 16; i++) s[0][i] = 0.f;
#pragma unroll
            for (uint32_t j = 0; j < DT; j++) {   // S^T += K Q^T
                wait_copies<4 * (DT - 1)>();
                // (products past the head are left out: a row of V may still lie there, and 0 times an infinity is not 0)
                const uint32_t n = j + 1 < DT ? 4u : (hb - 128 * j) / 32;
#pragma unroll
                for (uint32_t st = 0; st < 4; st++)
                    if (st < n) s[0] = mma16<float>(*reinterpret_cast<const i4v *>(lds + ka[st] + PIECE * j), q[4 * j + st], s[0]);
                wait_lds();
                copy(key, DT + j);
            }
            if (decltype(masked)::value) WaveAttn<_Float16, D>::hide(s[0], key, lim, lane);
            online_softmax<float>(s, o, m, l, c);
#pragma unroll
            for (uint32_t j = 0; j < DT; j++) {   // O^T += V^T P^T
                if (more) wait_copies<4 * (DT - 1)>();
                else wait_copies<0>();
                if (decltype(masked)::value) dropped |= drop_not_finite<float, 4>(lds + PIECE * j, lane);
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float a = *reinterpret_cast<const float *>(lds + va[i % 4 / 2] + PIECE * j + 128 * (8 * (i / 4) + i % 4));
                    o[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[0][i], o[j], 0, 0, 0);
                }
                wait_lds();
                if (more) copy(key + step, j);
            }
        };
        for (; key + 32 <= lim_all; key += step) subtile(std::false_type{});
        for (; key < k1; key += step) subtile(std::true_type{});
        return dropped;
    }
};

// Keys k0 .. k1 - 1 of some rows: a slot sees those below lim (each lane's own), every
// slot those below lim_all.
struct Span {
    Rows K, V;
    uint32_t k0, k1, lim, lim_all;
};

// ---- a workgroup: NW waves share 32 slots and take the spans' subtiles in turn
template <typename T, uint32_t D, uint32_t N>
struct BlockAttn {
    using W = WaveAttn<T, D>;
    static constexpr uint32_t NW = 4;
    // waves a SIMD that the LDS has room for: the registers are to allow them too
    static constexpr uint32_t WAVES = W::LDS <= 8192 ? (N > 1 ? 3 : 4) : W::LDS <= 12288 ? 3 : W::LDS <= 16384 ? 2 : 1;
    struct Shared {
        __align__(1024) uint8_t tiles[NW][W::LDS];
        float m[NW][32], l[NW][32];
        uint32_t lim[N][32], dropped[NW];
    };

    // out(slot of 32, dim, four sums, maximum, weight): joined over the waves
    template <typename OUT>
    __device__ __forceinline__ static void run(Shared &sh, const uint8_t *qrow, const Span (&sp)[N], uint32_t hb, float c,
                                               OUT out) {
        const uint32_t tid = threadIdx.x, lane = tid & 63u, h = lane >> 5, r32 = lane & 31u;
        const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        W w;
        w.init(qrow, hb, h);
        bool dropped = false;
        uint32_t turn = wave;   // the wave's first subtile of a span
#pragma unroll
        for (uint32_t n = 0; n < N; n++) {
            const Span &x = sp[n];
            dropped |= w.walk(x.K, x.V, hb, x.k0 + 32 * turn, 32 * NW, x.k1, x.lim, x.lim_all < x.k1 ? x.lim_all : x.k1,
                              sh.tiles[wave], lane, c);
            turn = (turn - (x.k1 - x.k0 + 31) / 32) % NW;
            if (h == 0) sh.lim[n][r32] = x.lim;   // (the same from every wave)
        }
        const float l = w.l + __shfl_xor(w.l, 32, 64);
        if (h == 0) {
            sh.m[wave][r32] = w.m;
            sh.l[wave][r32] = l;
        }
        if (lane == 0) sh.dropped[wave] = dropped;
        // the wave's subtiles make room for its sums, f32 [32][D], chunks XORed with the row (the writes of
        // eight lanes lie in different banks)
        uint8_t *const ob = sh.tiles[wave];
#pragma unroll
        for (uint32_t t = 0; t < W::DT; t++)
#pragma unroll
            for (uint32_t a = 0; a < 4; a++)
                *reinterpret_cast<f4v *>(ob + r32 * D * 4 + (((8 * t + 2 * a + h) ^ (r32 & 7u)) << 4)) =
                    f4v{w.o[t][4 * a], w.o[t][4 * a + 1], w.o[t][4 * a + 2], w.o[t][4 * a + 3]};
        __syncthreads();
        uint32_t any = 0;
#pragma unroll
        for (uint32_t x = 0; x < NW; x++) any |= sh.dropped[x];
        for (uint32_t i = tid; i < 32 * (D / 4); i += 64 * NW) {
            const uint32_t r = i / (D / 4), ch = i % (D / 4);
            float M = sh.m[0][r];
#pragma unroll
            for (uint32_t x = 1; x < NW; x++) M = fmaxf(M, sh.m[x][r]);
            float L = 0.f;
            f4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t x = 0; x < NW; x++) {
                // (a wave that saw no key of the slot has zeros, and m = -inf)
                const float f = sh.m[x][r] == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(sh.m[x][r] - M);
                const f4v o = *reinterpret_cast<const f4v *>(sh.tiles[x] + r * D * 4 + ((ch ^ (r & 7u)) << 4));
                L += f * sh.l[x][r];
                acc += f * o;
            }
            // (dropped from the first subtile on that some slot does not see whole)
            if (any && 4 * ch * W::SZ < hb) {
#pragma unroll
                for (uint32_t n = 0; n < N; n++) {
                    const Span &x = sp[n];
                    const uint32_t whole = x.lim_all < x.k1 ? x.lim_all : x.k1;
                    acc = add_not_finite<T>(acc, x.V.p + 4 * ch * W::SZ, x.V.stride, whole < x.k0 ? x.k0 : whole - (whole - x.k0) % 32,
                                            sh.lim[n][r]);
                }
            }
            out(r, 4 * ch, acc, M, L);
        }
    }
};

// ---- a workgroup of four waves with 32 slots each over tiles of keys that they
// share (16-bit types): tiles of NSUB subtiles, the next one's K and V on their
// way into the other half of the LDS while this one is worked on.  KS 2: eight
// waves, four of which take every other tile, and a join in LDS at the end: half
// the way through the keys where there are few workgroups.
template <typename T, uint32_t D, uint32_t KS>
struct TileAttn {
    using W = WaveAttn<T, D>;
    static constexpr uint32_t NW = 4, NSUB = W::SUB <= 8192 ? 2 : 1, TILE = NSUB * W::SUB, KEYS = 32 * NSUB;
    static constexpr uint32_t NC = NSUB * W::NL / NW;   // copies of a wave per tile of K, and of V
    static_assert(NSUB * W::NL % NW == 0);
    struct Shared {
        __align__(1024) uint8_t kv[KS][2][2][TILE];
        float m[NW][64], l[NW][64];   // (KS 2)
        uint32_t dropped[KS * NW];
    };
    static_assert(KS == 1 || sizeof(Shared::kv) >= NW * 32 * D * 4);

    // Keys k0 .. k1 - 1 of the workgroup, every slot of which sees those below
    // lim_all; the wave's slots see keys below lim (each lane's own), all of them
    // those below lim_lo, none those from lim_hi (0: the wave has no slots).
    // out(LDS of the wave, sums, maximum, weight).
    template <typename OUT>
    __device__ __forceinline__ static void run(Shared &sh, const uint8_t *qrow, const Rows &K, const Rows &V, uint32_t hb,
                                               uint32_t k0, uint32_t k1, uint32_t lim, uint32_t lim_all, uint32_t lim_lo,
                                               uint32_t lim_hi, float c, OUT out) {
        constexpr uint32_t RB = W::RB, C = W::C, SUB = W::SUB;
        const uint32_t tid = threadIdx.x, lane = tid & 63u, h = lane >> 5;
        const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6) % NW, ks = KS > 1 ? __builtin_amdgcn_readfirstlane(tid >> 6) / NW : 0u;
        auto &kv = sh.kv[ks];
        const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((lds_b)&kv[0][0][0]) + 1024 * NC * wave;
        W w;
        w.init(qrow, hb, h);
        if (hb < RB) {   // chunks past the head stay zero: copies leave them out
            for (uint32_t i = tid; i < sizeof(sh.kv) / 16; i += 64 * NW * KS)
                *reinterpret_cast<i4v *>(&sh.kv[0][0][0][0] + 16 * i) = i4v{0, 0, 0, 0};
            wait_lds();
            __builtin_amdgcn_s_barrier();
        }
        // this lane's part of its wave's copies: LDS chunk 64 (NC wave + i) + lane of the tile
        uint32_t off[2][NC];
#pragma unroll
        for (uint32_t i = 0; i < NC; i++) {
            const uint32_t L = 64 * (NC * wave + i) + lane, r = L / C;
            const uint32_t kc = 16 * ((L % C) ^ swizzle<C, 1>(r)), vc = 16 * ((L % C) ^ swizzle<C, 2>(r));
            off[0][i] = kc < hb ? r * K.stride + kc : ~0u;
            off[1][i] = vc < hb ? r * V.stride + vc : ~0u;
        }
        // K's tile at `at` (is_v 0) or V's into half `buf` of the LDS
        auto copy = [&](uint32_t is_v, uint32_t at, uint32_t buf) {
            const Rows &R = is_v ? V : K;
            const uint8_t *base = uniform(reinterpret_cast<uint64_t>(R.p) + (uint64_t)at * R.stride);
            const uint32_t dst = lds0 + TILE * (2 * buf + is_v);
            if (k1 - at >= KEYS && hb == RB) {
#pragma unroll
                for (uint32_t i = 0; i < NC; i++) copy_to_lds(base, off[is_v][i], dst + 1024 * i);
            } else if (k1 - at >= KEYS) {
#pragma unroll
                for (uint32_t i = 0; i < NC; i++)
                    if (off[is_v][i] != ~0u) copy_to_lds(base, off[is_v][i], dst + 1024 * i);
            } else {   // rows past the last key repeat it (hidden)
                const uint32_t last = k1 - at - 1u;
#pragma unroll
                for (uint32_t i = 0; i < NC; i++) {
                    const uint32_t L = 64 * (NC * wave + i) + (opaque(lane) & 63u), r = L / C, rr = r < last ? r : last;
                    const uint32_t ch = 16 * ((L % C) ^ (is_v ? swizzle<C, 2>(r) : swizzle<C, 1>(r)));
                    if (ch < hb) copy_to_lds(base, rr * R.stride + ch, dst + 1024 * i);
                }
            }
        };
        // The scores of the next tile are formed while this one's become weights and
        // meet V: products and vector instructions of one wave overlap then, and not
        // only those of the two waves of a SIMD.  K is a tile ahead of V for that.
        constexpr uint32_t STEP = KEYS * KS;
        uint32_t buf = 0, key = k0 + KEYS * ks;
        bool dropped = false;
        f16v s[NSUB];
        auto scores = [&](uint32_t half) {
#pragma unroll
            for (uint32_t n = 0; n < NSUB; n++) s[n] = w.scores(&kv[half][0][n * SUB], lane);
        };
        auto meet = [&]() {   // every wave's copies are there, and nobody reads what the next ones replace
            wait_lds();
            __builtin_amdgcn_s_barrier();
            __atomic_signal_fence(__ATOMIC_SEQ_CST);
        };
        if (key < k1) {
            copy(0, key, 0);
            copy(1, key, 0);
        }
        const bool two = key + STEP < k1;
        if (two) copy(0, key + STEP, 1);
        w.wait_queries();
        if (two) wait_copies<2 * NC>();
        else wait_copies<NC>();   // (none at all: nothing to wait for)
        meet();
        if (lim_hi > key) scores(0);
        // A whole tile's copies between the products, one after every fourth: the
        // four waves' copies take the memory unit 500 cycles, which they would
        // otherwise spend waiting for it right after they have met.
        static_assert(NSUB * W::NS == 4 * NC && NSUB * 2 * W::DT == 4 * NC);
        uint32_t steady = hb == RB && k1 >= 2 * STEP + KEYS ? k1 - 2 * STEP - KEYS + 1 : 0u;   // keys below: whole tiles two steps on
        steady = steady < lim_lo ? steady : lim_lo;
        for (; key < steady && key + KEYS <= lim_lo && key + KEYS <= lim_all; key += STEP, buf ^= 1u) {
            wait_copies<0>();
            meet();
            const uint8_t *kb = uniform(reinterpret_cast<uint64_t>(K.p) + (uint64_t)(key + 2 * STEP) * K.stride);
            const uint8_t *vb = uniform(reinterpret_cast<uint64_t>(V.p) + (uint64_t)(key + STEP) * V.stride);
            const uint32_t kd = lds0 + TILE * (2 * buf), vd = lds0 + TILE * (2 * (buf ^ 1u) + 1);
            new_maximum<T>(s, w.o, w.m, w.l, c);
            f16v p[NSUB];
#pragma unroll
            for (uint32_t n = 0; n < NSUB; n++) p[n] = s[n];
#pragma unroll
            for (uint32_t n = 0; n < NSUB; n++)
                s[n] = w.scores(&kv[buf ^ 1u][0][n * SUB], lane, [&](uint32_t st) {
                    const uint32_t i = n * W::NS + st;
                    if (i % 4 == 1) copy_to_lds(kb, off[0][i / 4], kd + 1024 * (i / 4));
                });
            weights(p, w.m, w.l, c);
#pragma unroll
            for (uint32_t n = 0; n < NSUB; n++)
                w.values(p[n], &kv[buf][1][n * SUB], lane, [&](uint32_t x) {
                    const uint32_t i = n * 2 * W::DT + x;
                    if (i % 4 == 1) copy_to_lds(vb, off[1][i / 4], vd + 1024 * (i / 4));
                });
        }
        auto next = [&]() {   // this tile's V and the next one's K are there, the ones after them on their way
            wait_copies<0>();
            if (key + KEYS > lim_all && key < k1)   // (each wave looks at what it copied)
                dropped |= drop_not_finite<T, NC>(&kv[buf][1][0] + 1024 * NC * wave, lane);
            meet();
            if (key + 2 * STEP < k1) copy(0, key + 2 * STEP, buf);
            if (key + STEP < k1) copy(1, key + STEP, buf ^ 1u);
        };
        for (; key + KEYS <= lim_lo; key += STEP, buf ^= 1u) {   // tiles that every slot of the wave sees whole
            next();
            new_maximum<T>(s, w.o, w.m, w.l, c);
            f16v p[NSUB];
#pragma unroll
            for (uint32_t n = 0; n < NSUB; n++) p[n] = s[n];
            scores(buf ^ 1u);   // (past the last tile: of what the LDS holds, and not looked at)
            weights(p, w.m, w.l, c);
#pragma unroll
            for (uint32_t n = 0; n < NSUB; n++) w.values(p[n], &kv[buf][1][n * SUB], lane);
        }
        // and the others; as many meetings for every wave
        for (; key < k1 + KEYS * ks; key += STEP, buf ^= 1u) {
            next();
            if (key >= lim_hi) continue;
#pragma unroll
            for (uint32_t n = 0; n < NSUB; n++) W::hide(s[n], key + 32 * n, lim, lane);
            new_maximum<T>(s, w.o, w.m, w.l, c);
            weights(s, w.m, w.l, c);
            const uint32_t ln = opaque(lane) & 63u;
#pragma unroll
            for (uint32_t n = 0; n < NSUB; n++) w.values(s[n], &kv[buf][1][n * SUB], ln);
            if (key + STEP < lim_hi) scores(buf ^ 1u);
        }
        float l = w.l + __shfl_xor(w.l, 32, 64), M = w.m;
        if (lane == 0) sh.dropped[NW * ks + wave] = dropped;
        __syncthreads();
        uint32_t any = 0;
#pragma unroll
        for (uint32_t i = 0; i < KS * NW; i++) any |= sh.dropped[i];
        if constexpr (KS > 1) {   // the other waves' sums to the first four, as the lanes hold them
            f4v *const ob = reinterpret_cast<f4v *>(&sh.kv[0][0][0][0]) + 8 * D * wave + lane;
            if (ks) {
                sh.m[wave][lane] = M;
                sh.l[wave][lane] = l;
#pragma unroll
                for (uint32_t t = 0; t < W::DT; t++)
#pragma unroll
                    for (uint32_t a = 0; a < 4; a++)
                        ob[64 * (4 * t + a)] = f4v{w.o[t][4 * a], w.o[t][4 * a + 1], w.o[t][4 * a + 2], w.o[t][4 * a + 3]};
            }
            __syncthreads();
            if (ks) return;
            const float m1 = sh.m[wave][lane], l1 = sh.l[wave][lane], mn = fmaxf(M, m1);
            // (no key of the slot: zeros, and a maximum of -inf)
            const float f0 = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(M - mn), f1 = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m1 - mn);
            M = mn;
            l = l * f0 + l1 * f1;
#pragma unroll
            for (uint32_t t = 0; t < W::DT; t++)
#pragma unroll
                for (uint32_t a = 0; a < 4; a++) {
                    const f4v x = ob[64 * (4 * t + a)];
#pragma unroll
                    for (int e = 0; e < 4; e++) w.o[t][4 * a + e] = w.o[t][4 * a + e] * f0 + x[e] * f1;
                }
        }
        if (any) {   // (dropped from the first tile on that some slot of the workgroup does not see whole)
#pragma unroll
            for (uint32_t t = 0; t < W::DT; t++)
#pragma unroll
                for (uint32_t a = 0; a < 4; a++) {
                    const uint32_t d = 32 * t + 8 * a + 4 * h;
                    f4v o = {w.o[t][4 * a], w.o[t][4 * a + 1], w.o[t][4 * a + 2], w.o[t][4 * a + 3]};
                    if (d * W::SZ < hb)
                        o = add_not_finite<T>(o, V.p + d * W::SZ, V.stride, lim_all < k0 ? k0 : lim_all - (lim_all - k0) % KEYS, lim);
#pragma unroll
                    for (int e = 0; e < 4; e++) w.o[t][4 * a + e] = o[e];
                }
        }
        // (KS 2: where this wave has just read its partner's sums)
        out(&sh.kv[0][0][0][0] + (KS > 1 ? 128 * D : sizeof(sh.kv) / NW) * wave, w.o, M, l);
    }
};

// four results of a row, rounded once to its type
template <typename T>
__device__ __forceinline__ void store4(uint8_t *row, uint32_t d, f4v x) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f4v *>(row + 4 * d) = x;
    } else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<t4 *>(row + 2 * d) = t4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
    }
}

// The wave's slots' rows, whole lines at a time: o as the lanes hold it through the
// wave's part of the LDS.  Straight from the registers a store would touch 32 rows
// for 16 bytes each (20 prompts of 100 rows, bf16: 20.9 us, so 18.5).  row: this
// lane's slot's (lane and lane + 32 the same), null if it has none; hb: bytes of
// the head.
template <typename T, uint32_t D>
__device__ __forceinline__ void store_rows(uint8_t *lds, const f16v (&o)[D / 32], float inv, uint8_t *row, uint32_t hb, uint32_t lane) {
    constexpr uint32_t C = D * sizeof(T) / 16;
    const uint32_t r32 = lane & 31u, h = lane >> 5;
#pragma unroll
    for (uint32_t t = 0; t < D / 32; t++)
#pragma unroll
        for (uint32_t a = 0; a < 4; a++) {
            const uint32_t byte = (32 * t + 8 * a + 4 * h) * sizeof(T);
            const f4v v = {o[t][4 * a], o[t][4 * a + 1], o[t][4 * a + 2], o[t][4 * a + 3]};
            store4<T>(lds + r32 * (16 * C) + (((byte >> 4) ^ swizzle<C, 1>(r32)) << 4) + (byte & 15u), 0, v * inv);
        }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);   // (other lanes' values next; a wave's LDS accesses are in order)
    const uint64_t at = reinterpret_cast<uint64_t>(row);
#pragma unroll
    for (uint32_t i = 0; i < 32 * C / 64; i++) {
        const uint32_t L = 64 * i + lane, r = L / C, ch = L % C;
        const i4v v = *reinterpret_cast<const i4v *>(lds + r * (16 * C) + ((ch ^ swizzle<C, 1>(r)) << 4));
        const uint64_t to = (uint64_t)(uint32_t)__shfl((int)(at >> 32), (int)r, 64) << 32 | (uint32_t)__shfl((int)(uint32_t)at, (int)r, 64);
        if (to && 16 * ch < hb) *reinterpret_cast<i4v *>(to + 16 * ch) = v;
    }
}

struct HeadShape {
    uint32_t group, n_kv, hd;   // query heads per KV head, KV heads, dims
    float c;                    // log2(e) / sqrt(hd)
};

// ---- packed prompts
struct PromptArgs {
    const uint8_t *q, *k, *v;
    uint8_t *out;
    uint32_t qs, ks, vs, os;    // bytes between rows
    const uint32_t *off;
    uint32_t n_seqs, n_rows;
    HeadShape s;
};

// Query tile y of the batch: its sequence's first row and length, and the tile
// inside it (tiles of a sequence from the last, with the most keys, to the
// first).  Offsets are the caller's data on the device: rows are clamped to the
// buffers'.  False past the last tile.
template <uint32_t SLOTS>
__device__ __forceinline__ bool find_tile(const uint32_t *off, uint32_t n_seqs, uint32_t n_rows, uint32_t group,
                                          uint32_t y, uint32_t lane, uint32_t *row0, uint32_t *len, uint32_t *tile) {
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < n_seqs; s0 += 64) {
        const uint32_t s = s0 + lane;
        uint32_t b = 0, e = 0;
        if (s < n_seqs) {
            b = off[s];
            e = off[s + 1];
            b = b < n_rows ? b : n_rows;
            e = e < n_rows ? e : n_rows;
            e = e > b ? e : b;
        }
        const uint32_t mine = ((e - b) * group + SLOTS - 1) / SLOTS;
        uint32_t sum = mine;   // inclusive over the lanes, by DPP row shifts and row broadcasts
        sum += __builtin_amdgcn_update_dpp(0, (int)sum, 0x111, 0xf, 0xf, false);
        sum += __builtin_amdgcn_update_dpp(0, (int)sum, 0x112, 0xf, 0xf, false);
        sum += __builtin_amdgcn_update_dpp(0, (int)sum, 0x114, 0xf, 0xf, false);
        sum += __builtin_amdgcn_update_dpp(0, (int)sum, 0x118, 0xf, 0xf, false);
        sum += __builtin_amdgcn_update_dpp(0, (int)sum, 0x142, 0xa, 0xf, false);
        sum += __builtin_amdgcn_update_dpp(0, (int)sum, 0x143, 0xc, 0xf, false);
        const uint64_t here = __ballot(before + sum > y);
        if (here) {
            const int at = __builtin_ctzll(here);
            *row0 = __builtin_amdgcn_readlane(b, at);
            *len = __builtin_amdgcn_readlane(e - b, at);
            *tile = before + __builtin_amdgcn_readlane(sum, at) - 1u - y;
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

template <typename T, uint32_t D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(BlockAttn<T, D, 1>::WAVES))) void prompt_attn_kernel(PromptArgs a) {
    using B = BlockAttn<T, D, 1>;
    __shared__ typename B::Shared sh;
    const uint32_t kvh = blockIdx.x % a.s.n_kv, lane = threadIdx.x & 63u;
    uint32_t row0, len, tile;
    if (!find_tile<kAttnTileRows>(a.off, a.n_seqs, a.n_rows, a.s.group, blockIdx.x / a.s.n_kv, lane, &row0, &len, &tile)) return;
    const uint32_t slots = len * a.s.group, slot0 = tile * kAttnTileRows, hb = a.s.hd * sizeof(T);
    const uint32_t last = (slot0 + kAttnTileRows < slots ? slot0 + kAttnTileRows : slots) - 1u;
    auto at = [&](uint32_t slot, uint32_t stride) {   // the slot's bytes in q or out
        const uint32_t r = slot / a.s.group;
        return (size_t)(row0 + r) * stride + (size_t)(kvh * a.s.group + (slot - r * a.s.group)) * hb;
    };
    const uint32_t mine = slot0 + (lane & 31u) < last ? slot0 + (lane & 31u) : last;
    const Rows K = {a.k + (size_t)row0 * a.ks + (size_t)kvh * hb, a.ks}, V = {a.v + (size_t)row0 * a.vs + (size_t)kvh * hb, a.vs};
    const Span seen[1] = {{K, V, 0, last / a.s.group + 1u, mine / a.s.group + 1u, slot0 / a.s.group + 1u}};
    B::run(sh, a.q + at(mine, a.qs), seen, hb, a.s.c, [&](uint32_t r, uint32_t d, f4v o, float, float L) {
        if (slot0 + r <= last && d < a.s.hd) store4<T>(a.out + at(slot0 + r, a.os), d, o * (L == 0.f ? 0.f : 1.0f / L));
    });
}

// the same by workgroups of 128 slots
template <typename T, uint32_t D, uint32_t KS>
__global__ __launch_bounds__(256 * KS) __attribute__((amdgpu_waves_per_eu(D <= 128 || KS > 1 ? 2 : 1))) void prompt_tile_kernel(PromptArgs a) {
    using B = TileAttn<T, D, KS>;
    __shared__ typename B::Shared sh;
    const uint32_t kvh = blockIdx.x % a.s.n_kv, lane = threadIdx.x & 63u, g = a.s.group;
    uint32_t row0, len, tile;
    if (!find_tile<128>(a.off, a.n_seqs, a.n_rows, g, blockIdx.x / a.s.n_kv, lane, &row0, &len, &tile)) return;
    const uint32_t hb = a.s.hd * sizeof(T), end = len * g - 1u, slot0 = 128 * tile;
    const uint32_t last = slot0 + 127 < end ? slot0 + 127 : end;   // the workgroup's last slot
    const uint32_t first_w = slot0 + 32 * (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3u);
    const uint32_t last_w = first_w + 31 < last ? first_w + 31 : last, mine = first_w + (lane & 31u) < last ? first_w + (lane & 31u) : last;
    const uint32_t r = mine / g;
    const size_t head = (size_t)(kvh * g + (mine - r * g)) * hb;
    const Rows K = {a.k + (size_t)row0 * a.ks + (size_t)kvh * hb, a.ks}, V = {a.v + (size_t)row0 * a.vs + (size_t)kvh * hb, a.vs};
    const bool any = first_w <= last, own = first_w + (lane & 31u) <= last;
    uint8_t *const out = own ? a.out + (size_t)(row0 + r) * a.os + head : nullptr;
    B::run(sh, a.q + (size_t)(row0 + r) * a.qs + head, K, V, hb, 0, last / g + 1u, r + 1u, slot0 / g + 1u, any ? first_w / g + 1u : 0u,
           any ? last_w / g + 1u : 0u, a.s.c, [&](uint8_t *lds, f16v (&o)[D / 32], float, float L) {
               store_rows<T, D>(lds, o, L == 0.f ? 0.f : 1.0f / L, out, hb, lane);
           });
}

// ---- new tokens over a shared prefix and their own tails
struct PrefixArgs {
    const uint8_t *q, *kp, *vp, *kt, *vt;
    uint32_t qs, kps, vps, kts, vts;
    const uint32_t *lens;
    uint32_t prefix, cap, n_seqs, n_tokens;
    uint32_t p_chunk, n_p, p_tiles, t_chunk, n_t, t_tiles, p_jobs;   // (p_jobs: of one KV head)
    float2 *ml;   // [chunk][row][head]
    float *o;     // [chunk][row][head][hd]
    HeadShape s;
};

// TILE: the prefix by workgroups of 128 slots that share its tiles
template <typename T, uint32_t D, bool TILE>
__global__ __launch_bounds__(256)
    __attribute__((amdgpu_waves_per_eu(TILE ? (D <= 128 ? 2 : 1) : BlockAttn<T, D, 1>::WAVES))) void prefix_attn_kernel(PrefixArgs a) {
    using B = BlockAttn<T, D, 1>;
    using P = TileAttn<typename std::conditional<TILE, T, _Float16>::type, TILE ? D : 64, 1>;
    __shared__ union {
        typename B::Shared block;
        typename std::conditional<TILE, typename P::Shared, char>::type tile;
    } sh;
    const uint32_t lane = threadIdx.x & 63u, hb = a.s.hd * sizeof(T), g = a.s.group, n_heads = g * a.s.n_kv;
    const uint32_t kvh = blockIdx.x % a.s.n_kv, n_rows = a.n_seqs * a.n_tokens;
    uint32_t job = blockIdx.x / a.s.n_kv, row0 = 0;
    auto pair = [&](uint32_t slot) {   // (row, head) of the slot
        const uint32_t r = slot / g;
        return (size_t)(row0 + r) * n_heads + kvh * g + (slot - r * g);
    };
    auto query = [&](uint32_t slot) {
        const uint32_t r = slot / g;
        return a.q + (size_t)(row0 + r) * a.qs + (size_t)(kvh * g + (slot - r * g)) * hb;
    };
    if (job < a.p_jobs) {
        const uint32_t tile = job % a.p_tiles, chunk = job / a.p_tiles, slots = n_rows * g;
        const uint32_t k0 = chunk * a.p_chunk, k1 = a.prefix - k0 < a.p_chunk ? a.prefix : k0 + a.p_chunk;
        const Rows K = {a.kp + (size_t)kvh * hb, a.kps}, V = {a.vp + (size_t)kvh * hb, a.vps};
        const size_t part = (size_t)chunk * n_rows * n_heads;
        if constexpr (TILE) {
            const uint32_t first = 128 * tile + 32 * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = first + (lane & 31u);
            const uint32_t mine = slot < slots ? slot : slots - 1u;
            const size_t at = part + pair(mine);
            P::run(sh.tile, query(mine), K, V, hb, k0, k1, k1, k1, first < slots ? k1 : 0u, first < slots ? k1 : 0u, a.s.c,
                   [&](uint8_t *, f16v (&o)[D / 32], float M, float L) {
                       if (slot >= slots) return;
                       if (lane < 32) a.ml[at] = make_float2(M, L);
#pragma unroll
                       for (uint32_t t = 0; t < D / 32; t++)
#pragma unroll
                           for (uint32_t x = 0; x < 4; x++) {
                               const uint32_t d = 32 * t + 8 * x + 4 * (lane >> 5);
                               if (d < a.s.hd)
                                   *reinterpret_cast<f4v *>(a.o + at * a.s.hd + d) = f4v{o[t][4 * x], o[t][4 * x + 1], o[t][4 * x + 2], o[t][4 * x + 3]};
                           }
                   });
        } else {
            const uint32_t slot0 = tile * kAttnTileRows, slot = slot0 + (lane & 31u);
            const Span seen[1] = {{K, V, k0, k1, k1, k1}};
            B::run(sh.block, query(slot < slots ? slot : slots - 1u), seen, hb, a.s.c,
                   [&](uint32_t i, uint32_t d, f4v o, float M, float L) {
                       if (slot0 + i >= slots || d >= a.s.hd) return;
                       const size_t at = part + pair(slot0 + i);
                       if (d == 0) a.ml[at] = make_float2(M, L);
                       *reinterpret_cast<f4v *>(a.o + at * a.s.hd + d) = o;
                   });
        }
        return;
    }
    job -= a.p_jobs;
    const uint32_t tile = job % a.t_tiles;
    job /= a.t_tiles;
    const uint32_t seq = job % a.n_seqs, len = a.lens[seq] < a.cap ? a.lens[seq] : a.cap, chunk = job / a.n_seqs;
    row0 = seq * a.n_tokens;
    const uint32_t slots = a.n_tokens * g, slot0 = tile * kAttnTileRows;
    const uint32_t last = slot0 + kAttnTileRows < slots ? slot0 + kAttnTileRows - 1u : slots - 1u;
    const uint32_t mine = slot0 + (lane & 31u) < last ? slot0 + (lane & 31u) : last;
    // token i sees rows below len - n_tokens + 1 + i of the tail
    auto sees = [&](uint32_t slot) {
        const uint32_t n = len + 1u + slot / g;
        return n > a.n_tokens ? n - a.n_tokens : 0u;
    };
    const uint32_t k0 = chunk * a.t_chunk, k1 = sees(last) < k0 + a.t_chunk ? sees(last) : k0 + a.t_chunk;
    const size_t part = (size_t)(a.n_p + chunk) * n_rows * n_heads;
    if (k0 >= k1) {   // nothing of the tail in this chunk
        if (threadIdx.x < 32 && slot0 + threadIdx.x <= last) a.ml[part + pair(slot0 + threadIdx.x)] = make_float2(-INFINITY, 0.f);
        return;
    }
    const Rows K = {a.kt + (size_t)seq * a.cap * a.kts + (size_t)kvh * hb, a.kts};
    const Rows V = {a.vt + (size_t)seq * a.cap * a.vts + (size_t)kvh * hb, a.vts};
    const Span seen[1] = {{K, V, k0, k1, sees(mine) < k1 ? sees(mine) : k1, sees(slot0)}};
    B::run(sh.block, query(mine), seen, hb, a.s.c, [&](uint32_t i, uint32_t d, f4v o, float M, float L) {
        if (slot0 + i > last || d >= a.s.hd) return;
        const size_t at = part + pair(slot0 + i);
        if (d == 0) a.ml[at] = make_float2(M, L);
        *reinterpret_cast<f4v *>(a.o + at * a.s.hd + d) = o;
    });
}

// The same without chunks, in one launch: a workgroup walks the prefix and then its
// sequence's tail.
template <typename T, uint32_t D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(BlockAttn<T, D, 2>::WAVES))) void prefix_short_kernel(
    PrefixArgs a, uint8_t *out, uint32_t os) {
    using B = BlockAttn<T, D, 2>;
    __shared__ typename B::Shared sh;
    const uint32_t lane = threadIdx.x & 63u, hb = a.s.hd * sizeof(T), g = a.s.group, kvh = blockIdx.x % a.s.n_kv;
    const uint32_t job = blockIdx.x / a.s.n_kv, tile = job % a.t_tiles, seq = job / a.t_tiles;
    const uint32_t len = a.lens[seq] < a.cap ? a.lens[seq] : a.cap, row0 = seq * a.n_tokens;
    const uint32_t slots = a.n_tokens * g, slot0 = tile * kAttnTileRows;
    const uint32_t last = slot0 + kAttnTileRows < slots ? slot0 + kAttnTileRows - 1u : slots - 1u;
    const uint32_t mine = slot0 + (lane & 31u) < last ? slot0 + (lane & 31u) : last;
    auto sees = [&](uint32_t slot) {
        const uint32_t n = len + 1u + slot / g;
        return n > a.n_tokens ? n - a.n_tokens : 0u;
    };
    auto at = [&](uint32_t slot, uint32_t stride) {
        const uint32_t r = slot / g;
        return (size_t)(row0 + r) * stride + (size_t)(kvh * g + (slot - r * g)) * hb;
    };
    const Span seen[2] = {{{a.kp + (size_t)kvh * hb, a.kps}, {a.vp + (size_t)kvh * hb, a.vps}, 0, a.prefix, a.prefix, a.prefix},
                          {{a.kt + (size_t)seq * a.cap * a.kts + (size_t)kvh * hb, a.kts},
                           {a.vt + (size_t)seq * a.cap * a.vts + (size_t)kvh * hb, a.vts}, 0, sees(last), sees(mine), sees(slot0)}};
    B::run(sh, a.q + at(mine, a.qs), seen, hb, a.s.c, [&](uint32_t i, uint32_t d, f4v o, float, float L) {
        if (slot0 + i <= last && d < a.s.hd) store4<T>(out + at(slot0 + i, os), d, o * (L == 0.f ? 0.f : 1.0f / L));
    });
}

// out = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c over a row's chunks, a
// workgroup per (row, head): its threads take the chunks' factors together, then
// groups of G lanes (four dims each) take the chunks in turn, so that their
// loads do not wait for each other.  A row that saw no key has l = 0 everywhere
// and gives zeros.
template <typename T, uint32_t NT, uint32_t G, uint32_t AHEAD>
__global__ __launch_bounds__(NT) void prefix_join_kernel(const float2 *__restrict__ ml, const float *__restrict__ o,
                                                         uint8_t *__restrict__ out, uint32_t os, uint32_t rows,
                                                         uint32_t n_heads, uint32_t hd, uint32_t parts) {
    constexpr uint32_t NG = NT / G, NW = NT / 64;
    __shared__ float f[kMaxParts];   // a chunk's factor; -1: it saw no key, and its sums were not written
    __shared__ float red[2][NW];
    __shared__ f4v sums[NG][G];
    const uint32_t at = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, g = tid / G, d = 4 * (tid % G);
    // a group's first AHEAD sums are on their way while the factors are worked out
    const float *mine = o + (size_t)at * hd + (d < hd ? d : 0u);
    const size_t step = (size_t)rows * hd;
    f4v first[AHEAD + 1];
#pragma unroll
    for (uint32_t i = 0; i < AHEAD; i++) first[i] = *reinterpret_cast<const f4v *>(mine + (g + i * NG < parts ? g + i * NG : 0u) * step);
    float M = -INFINITY;
    for (uint32_t p = tid; p < parts; p += NT) M = fmaxf(M, ml[(size_t)p * rows + at].x);
#pragma unroll
    for (uint32_t x = 32; x; x /= 2) M = fmaxf(M, __shfl_xor(M, x, 64));
    if (NW > 1) {
        if (lane == 0) red[0][tid >> 6] = M;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < NW; w++) M = fmaxf(M, red[0][w]);
    }
    float L = 0.f;
    for (uint32_t p = tid; p < parts; p += NT) {
        const float2 x = ml[(size_t)p * rows + at];
        const bool none = x.x == -INFINITY && x.y == 0.f;
        const float e = none ? -1.f : __builtin_amdgcn_exp2f(x.x - M);
        f[p] = e;
        if (!none) L += e * x.y;
    }
#pragma unroll
    for (uint32_t x = 32; x; x /= 2) L += __shfl_xor(L, x, 64);
    if (lane == 0) red[1][tid >> 6] = L;
    __syncthreads();
    f4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t i = 0; i < AHEAD; i++) {
        const uint32_t p = g + i * NG;
        const float e = p < parts ? f[p] : -1.f;
        if (e != -1.f) acc += e * first[i];
    }
#pragma unroll 4
    for (uint32_t p = g + AHEAD * NG; p < parts; p += NG) {
        const float e = f[p];
        if (e != -1.f) acc += e * *reinterpret_cast<const f4v *>(mine + p * step);
    }
    sums[g][tid % G] = acc;
    __syncthreads();
    if (tid < G && d < hd) {
        L = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < NW; w++) L += red[1][w];
        acc = sums[0][tid];
#pragma unroll
        for (uint32_t i = 1; i < NG; i++) acc += sums[i][tid];
        const uint32_t row = at / n_heads;
        store4<T>(out + (size_t)row * os + (size_t)(at - row * n_heads) * hd * sizeof(T), d, acc * (L == 0.f ? 0.f : 1.0f / L));
    }
}

// f(element type, padded head size)
template <typename F>
static void by_shape(uint32_t dtype, uint32_t hd, F f) {
    auto dims = [&](auto t) {
        const uint32_t d = attn_padded_dim(hd, sizeof(t));
        if constexpr (sizeof(t) == 4) {
            switch (d) {
            case 32: f(t, std::integral_constant<uint32_t, 32>{}); return;
            case 160: f(t, std::integral_constant<uint32_t, 160>{}); return;
            case 192: f(t, std::integral_constant<uint32_t, 192>{}); return;
            case 224: f(t, std::integral_constant<uint32_t, 224>{}); return;
            }
        }
        switch (d) {
        case 64: f(t, std::integral_constant<uint32_t, 64>{}); break;
        case 96: f(t, std::integral_constant<uint32_t, 96>{}); break;
        case 128: f(t, std::integral_constant<uint32_t, 128>{}); break;
        default: f(t, std::integral_constant<uint32_t, 256>{}); break;
        }
    };
    if (dtype == YULE_DTYPE_F32) dims(float{});
    else if (dtype == YULE_DTYPE_F16) dims((_Float16)0);
    else dims((__bf16)0);
}

static HeadShape head_shape(uint32_t n_heads, uint32_t n_kv, uint32_t hd) {
    return {n_heads / n_kv, n_kv, hd, (float)(1.44269504088896340736 / sqrt((double)hd))};
}

static int launch_prompt(hipStream_t s, const PromptArgs &a, uint32_t dtype, const PromptPlan &p) {
    const dim3 grid((uint32_t)(p.tiles * a.s.n_kv));
    by_shape(dtype, a.s.hd, [&](auto t, auto d) {
        using T = decltype(t);
        constexpr uint32_t D = decltype(d)::value;
        if constexpr (sizeof(T) == 2) {
            if (p.slots == 128) {
                if constexpr (D <= 128) {
                    if (p.split == 2) {
                        hipLaunchKernelGGL((prompt_tile_kernel<T, D, 2>), grid, dim3(512), 0, s, a);
                        return;
                    }
                }
                hipLaunchKernelGGL((prompt_tile_kernel<T, D, 1>), grid, dim3(256), 0, s, a);
                return;
            }
        }
        hipLaunchKernelGGL((prompt_attn_kernel<T, D>), grid, dim3(256), 0, s, a);
    });
    return check_launch("prompt_attn");
}

static int launch_prefix(hipStream_t s, const PrefixArgs &a, uint32_t dtype, uint64_t workgroups, bool tile) {
    by_shape(dtype, a.s.hd, [&](auto t, auto d) {
        using T = decltype(t);
        constexpr uint32_t D = decltype(d)::value;
        if constexpr (sizeof(T) == 2) {
            if (tile) {
                hipLaunchKernelGGL((prefix_attn_kernel<T, D, true>), dim3((uint32_t)workgroups), dim3(256), 0, s, a);
                return;
            }
        }
        hipLaunchKernelGGL((prefix_attn_kernel<T, D, false>), dim3((uint32_t)workgroups), dim3(256), 0, s, a);
    });
    return check_launch("prefix_attn");
}

static int launch_prefix_short(hipStream_t s, const PrefixArgs &a, uint8_t *out, uint32_t os, uint32_t dtype) {
    const dim3 grid(a.s.n_kv * a.t_tiles * a.n_seqs);
    by_shape(dtype, a.s.hd, [&](auto t, auto d) {
        hipLaunchKernelGGL((prefix_short_kernel<decltype(t), decltype(d)::value>), grid, dim3(256), 0, s, a, out, os);
    });
    return check_launch("prefix_attn");
}

static int launch_join(hipStream_t s, const PrefixArgs &a, uint8_t *out, uint32_t os, uint32_t dtype) {
    const uint32_t n_heads = a.s.group * a.s.n_kv, rows = a.n_seqs * a.n_tokens * n_heads, hd = a.s.hd, parts = a.n_p + a.n_t;
    by_shape(dtype, hd, [&](auto t, auto d) {
        using T = decltype(t);
        constexpr uint32_t D = decltype(d)::value, G = D <= 64 ? 16 : D <= 128 ? 32 : 64;
        auto go = [&](auto nt, auto ahead) {
            constexpr uint32_t NT = decltype(nt)::value;
            hipLaunchKernelGGL((prefix_join_kernel<T, NT, G, decltype(ahead)::value>), dim3(rows), dim3(NT), 0, s, a.ml, a.o,
                               out, os, rows, n_heads, hd, parts);
        };
        using N = std::integral_constant<uint32_t, 0>;
        using One = std::integral_constant<uint32_t, 64>;
        using Four = std::integral_constant<uint32_t, 256>;
        // One wave where it takes every chunk in a step or two.  Loads ahead where a group has more than four chunks:
        // 60 of them, 156 rows: 12.7 us of the two launches against 14.7; 12 or 32 chunks, with as many loads for
        // nothing, 17.1 against 16.8 and 53.5 against 51.5.
        if (parts <= 2 * 64 / G) go(One{}, N{});
        else if (parts <= 4 * 256 / G) go(Four{}, N{});
        else go(Four{}, std::integral_constant<uint32_t, 8>{});
    });
    return check_launch("prefix_attn (join)");
}

// ---- C entries
namespace {

struct Checked {
    uint8_t *p;
    uint32_t stride;   // bytes
};

int rows_arg(yule_hip_backend *be, const yule_rows *r, uint64_t n_rows, uint64_t width, uint32_t elem, const char *what,
             Checked *out) {
    void *p;
    int rc = rows_ptr(be, r, n_rows, width, elem, 16, kMaxAttnStride, what, &p);
    if (rc) return rc;
    out->p = static_cast<uint8_t *>(p);
    out->stride = n_rows > 1 ? (uint32_t)(r->stride * elem) : 0u;   // (one row or none: any stride is given)
    return YULE_OK;
}

}  // namespace
}  // namespace yule

using namespace yule;

extern "C" {

int yule_hip_prompt_attn(yule_hip_backend *be, const yule_rows *q, const yule_rows *k, const yule_rows *v,
                         const yule_rows *out, yule_buffer offsets, uint32_t n_seqs, uint32_t n_rows, uint32_t n_heads,
                         uint32_t n_kv_heads, uint32_t head_dim, uint32_t dtype) {
    return guarded("prompt_attn", be, [&]() -> int {
        const uint32_t elem = attn_elem_bytes(dtype);
        if (!elem) return set_error(YULE_ERR_UNSUPPORTED, "prompt_attn: dtype " + std::to_string(dtype) + " not supported");
        if (const char *bad = check_heads(n_heads, n_kv_heads, head_dim))
            return set_error(YULE_ERR_INVALID, std::string("prompt_attn: ") + bad);
        const uint64_t qd = (uint64_t)n_heads * head_dim, kvd = (uint64_t)n_kv_heads * head_dim;
        Checked cq, ck, cv, co;
        void *off;
        int rc;
        if ((rc = rows_arg(be, q, n_rows, qd, elem, "prompt_attn (q)", &cq)) ||
            (rc = rows_arg(be, k, n_rows, kvd, elem, "prompt_attn (k)", &ck)) ||
            (rc = rows_arg(be, v, n_rows, kvd, elem, "prompt_attn (v)", &cv)) ||
            (rc = rows_arg(be, out, n_rows, qd, elem, "prompt_attn (out)", &co)) ||
            (rc = get_buffer(be, offsets, ((size_t)n_seqs + 1) * 4, &off, "prompt_attn (offsets)", 0, true)))
            return rc;
        if (out->buffer == q->buffer || out->buffer == k->buffer || out->buffer == v->buffer || out->buffer == offsets)
            return set_error(YULE_ERR_INVALID, "prompt_attn: an input and the output alias");
        if (!n_seqs || !n_rows) return YULE_OK;
        const PromptPlan p = prompt_plan(n_seqs, n_rows, n_heads, n_kv_heads, head_dim, elem, (uint32_t)be->props.multiProcessorCount);
        if ((uint64_t)n_rows * (n_heads / n_kv_heads) >= (uint64_t)1 << 31 || p.tiles * n_kv_heads > kMaxWorkgroups)
            return set_error(YULE_ERR_INVALID, "prompt_attn: too many rows for one call");
        const PromptArgs a = {cq.p, ck.p, cv.p, co.p, cq.stride, ck.stride, cv.stride, co.stride,
                              static_cast<const uint32_t *>(off), n_seqs, n_rows, head_shape(n_heads, n_kv_heads, head_dim)};
        return launch_prompt(be->stream, a, dtype, p);
    });
}

int yule_hip_prefix_attn(yule_hip_backend *be, const yule_rows *q, const yule_rows *k_prefix, const yule_rows *v_prefix,
                         uint32_t prefix_len, const yule_rows *k_tail, const yule_rows *v_tail, yule_buffer tail_lens,
                         uint32_t tail_cap, const yule_rows *out, uint32_t n_seqs, uint32_t n_tokens, uint32_t n_heads,
                         uint32_t n_kv_heads, uint32_t head_dim, uint32_t dtype) {
    return guarded("prefix_attn", be, [&]() -> int {
        const uint32_t elem = attn_elem_bytes(dtype);
        if (!elem) return set_error(YULE_ERR_UNSUPPORTED, "prefix_attn: dtype " + std::to_string(dtype) + " not supported");
        if (const char *bad = check_heads(n_heads, n_kv_heads, head_dim))
            return set_error(YULE_ERR_INVALID, std::string("prefix_attn: ") + bad);
        if (!n_tokens || n_tokens > 64) return set_error(YULE_ERR_INVALID, "prefix_attn: n_tokens must be 1..64");
        if (prefix_len > kMaxKeys || tail_cap > kMaxKeys)
            return set_error(YULE_ERR_INVALID, "prefix_attn: more than 2^30 keys");
        const uint64_t qd = (uint64_t)n_heads * head_dim, kvd = (uint64_t)n_kv_heads * head_dim;
        const uint64_t rows = (uint64_t)n_seqs * n_tokens, tails = (uint64_t)n_seqs * tail_cap;
        Checked cq, ckp = {}, cvp = {}, ckt = {}, cvt = {}, co;
        void *lens;
        int rc;
        if ((rc = rows_arg(be, q, rows, qd, elem, "prefix_attn (q)", &cq)) ||
            (prefix_len && ((rc = rows_arg(be, k_prefix, prefix_len, kvd, elem, "prefix_attn (k_prefix)", &ckp)) ||
                            (rc = rows_arg(be, v_prefix, prefix_len, kvd, elem, "prefix_attn (v_prefix)", &cvp)))) ||
            (tail_cap && ((rc = rows_arg(be, k_tail, tails, kvd, elem, "prefix_attn (k_tail)", &ckt)) ||
                          (rc = rows_arg(be, v_tail, tails, kvd, elem, "prefix_attn (v_tail)", &cvt)))) ||
            (rc = rows_arg(be, out, rows, qd, elem, "prefix_attn (out)", &co)) ||
            (rc = get_buffer(be, tail_lens, (size_t)n_seqs * 4, &lens, "prefix_attn (tail_lens)", 0, true)))
            return rc;
        if (out->buffer == q->buffer || out->buffer == tail_lens ||
            (prefix_len && (out->buffer == k_prefix->buffer || out->buffer == v_prefix->buffer)) ||
            (tail_cap && (out->buffer == k_tail->buffer || out->buffer == v_tail->buffer)))
            return set_error(YULE_ERR_INVALID, "prefix_attn: an input and the output alias");
        if (!n_seqs) return YULE_OK;
        const PrefixPlan p = prefix_plan(prefix_len, tail_cap, n_seqs, n_tokens, n_heads, n_kv_heads, head_dim, elem,
                                         (uint32_t)be->props.multiProcessorCount);
        if (p.rows > kMaxWorkgroups || p.p_jobs + p.t_jobs > kMaxWorkgroups)
            return set_error(YULE_ERR_INVALID, "prefix_attn: too many rows for one call");
        ScratchLease ws;   // held until both launches are enqueued
        if (!p.direct && (rc = get_scratch(be, p.bytes(), &ws))) return rc;
        PrefixArgs a = {};
        a.q = cq.p, a.kp = ckp.p, a.vp = cvp.p, a.kt = ckt.p, a.vt = cvt.p;
        a.qs = cq.stride, a.kps = ckp.stride, a.vps = cvp.stride, a.kts = ckt.stride, a.vts = cvt.stride;
        a.lens = static_cast<const uint32_t *>(lens);
        a.prefix = prefix_len, a.cap = tail_cap, a.n_seqs = n_seqs, a.n_tokens = n_tokens;
        a.p_chunk = p.p_chunk, a.n_p = p.n_p, a.p_tiles = p.p_tiles;
        a.t_chunk = p.t_chunk, a.n_t = p.n_t, a.t_tiles = p.t_tiles, a.p_jobs = (uint32_t)(p.p_jobs / n_kv_heads);
        a.s = head_shape(n_heads, n_kv_heads, head_dim);
        if (p.direct) return launch_prefix_short(be->stream, a, co.p, co.stride, dtype);
        a.ml = static_cast<float2 *>(ws.ptr);
        a.o = reinterpret_cast<float *>(static_cast<uint8_t *>(ws.ptr) + p.ml_bytes);
        if (p.p_jobs + p.t_jobs && (rc = launch_prefix(be->stream, a, dtype, p.p_jobs + p.t_jobs, p.p_slots > kAttnTileRows))) return rc;
        return launch_join(be->stream, a, co.p, co.stride, dtype);
    });
}

}  // extern "C"
