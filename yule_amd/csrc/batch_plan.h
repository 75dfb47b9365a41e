// batch_plan.h — what the batched serving operators decide on the host: the
// checks of their arguments, how work is split, and where results that are
// joined later lie in the workspace.  Plain C++ (no HIP), so that a program
// without a GPU can check it.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cstdio>

#include "../../include/yule_hip.h"

namespace yule {

// bytes of one element of an attention type; 0: not one
inline uint32_t attn_elem_bytes(uint32_t dtype) {
    return dtype == YULE_DTYPE_F32 ? 4u : dtype == YULE_DTYPE_F16 || dtype == YULE_DTYPE_BF16 ? 2u : 0u;
}

// the head size that the kernels are built for (dims past head_dim are zeros in
// registers, and zeros in LDS or left out); f32: the next multiple of 32, so that
// every piece of 32 dims holds some of the head
inline uint32_t attn_padded_dim(uint32_t hd, uint32_t elem) {
    return elem == 4 ? (hd + 31) / 32 * 32 : hd <= 64 ? 64u : hd <= 96 ? 96u : hd <= 128 ? 128u : 256u;
}

// Rows r < n_rows, each `width` elements of `elem` bytes, of a buffer of
// buf_bytes: nullptr, or what is wrong.  align: bytes that every row starts at
// a multiple of.  max_stride: of several rows, what every stride is below.
// Attention's: offsets inside a tile (32 rows of f32, 64 of 16-bit types) have to fit
// 31 bits, as the copies into LDS take 32-bit offsets from a 64-bit row address.
constexpr uint64_t kMaxAttnStride = (uint64_t)1 << 24, kAnyStride = ~(uint64_t)0;
inline const char *check_rows(uint64_t offset, uint64_t stride, uint64_t n_rows, uint64_t width, uint32_t elem,
                              uint64_t buf_bytes, uint32_t align, uint64_t max_stride = kMaxAttnStride) {
    if (!n_rows || !width) return nullptr;
    const uint64_t elems = buf_bytes / elem;
    if (stride < width && n_rows > 1) return "rows overlap (stride below the row's width)";
    if (stride >= max_stride && n_rows > 1) return "row stride of 2^24 elements or more";
    if (width > elems || offset > elems - width) return "rows reach past the buffer";
    if (n_rows > 1 && (elems - width - offset) / stride < n_rows - 1) return "rows reach past the buffer";
    if ((offset * elem) % align || (n_rows > 1 && (stride * elem) % align)) return "rows are not aligned";
    return nullptr;
}

// heads and types of an attention call: nullptr, or what is wrong
inline const char *check_heads(uint32_t n_heads, uint32_t n_kv, uint32_t hd) {
    if (!n_heads || !n_kv || n_heads % n_kv) return "n_heads must be a positive multiple of n_kv_heads";
    if (!hd || hd % 8 || hd > 256) return "head_dim must be a multiple of 8, at most 256";
    if (n_heads > 4096) return "more than 4096 heads";
    return nullptr;
}

// (query rows x heads per KV head) of one wave's tile
constexpr uint32_t kAttnTileRows = 32;
// workgroups of one launch: its threads count in 32 bits
constexpr uint64_t kMaxWorkgroups = (uint64_t)1 << 23;
constexpr uint32_t kMaxKeys = 1u << 30;   // of a prefix, and of a tail

// ---- prompt_attn: who takes a tile of (row, head of the group) pairs of a KV head.
// f32: a workgroup per 32 of them, its four waves share the keys.  16-bit types,
// by what was measured (MI355X, bf16, us; heads / KV heads x head_dim, rows):
//   32     the same, while all of them find room on the chip at once: latency
//          counts, and many small workgroups have the shortest way
//          (32/8x128: 128 rows 6.8 against 8.9 with 128, 500 rows 11.8 against
//          14.9; 750 rows, too many, 22.0 against 18.5; 32/4x64, 1000 rows: 14.1
//          against 15.6 and 17.4)
//   split  128 a workgroup of eight waves, half of which take every other tile of
//          keys: few workgroups with a long way (32/8x128: 1000 rows 21.8 against
//          23.3, but 2000 rows, twice the workgroups, 47.1 against 45.8; 12/2x80,
//          3000 rows: 40.8 against 51.5; but seven sequences of 259 rows on
//          average 28.1 against 22.9)
//   128    four waves of 32 over shared tiles of keys: throughput
struct PromptPlan {
    uint32_t slots, split;   // pairs of a tile, groups of waves that share its keys
    uint64_t tiles;          // at most: each sequence has one that is not full
};
// workgroups of the 32-pair kernel that a CU's LDS has room for
inline uint32_t attn_block_room(uint32_t hd, uint32_t elem) {
    const uint32_t d = attn_padded_dim(hd, elem), lds = 4 * (elem == 4 ? 128 * d : 64 * d * elem) + 2048;
    return 163840u / lds;
}
inline PromptPlan prompt_plan(uint32_t n_seqs, uint32_t n_rows, uint32_t n_heads, uint32_t n_kv, uint32_t hd,
                              uint32_t elem, uint32_t cus) {
    const uint64_t pairs = (uint64_t)n_rows * (n_heads / n_kv), small = pairs / 32 + n_seqs, large = pairs / 128 + n_seqs;
    if (elem == 4 || small * n_kv <= (uint64_t)attn_block_room(hd, elem) * cus) return {32, 1, small};
    const bool split = 2 * large * n_kv <= 3ull * cus && n_rows / n_seqs >= 512 && hd <= 128;
    return {128, split ? 2u : 1u, large};
}

// ---- verify_drafts: values of a row that a workgroup takes
constexpr uint32_t kVerifyChunk = 4096, kMaxVocab = 1u << 30, kMaxDrafts = 1024;
// sequences of one launch, and words between their tickets: a line of 128 bytes
// each (512 workgroups that draw from one line queue for it: 16 rows of 128256
// values 15.1 us, with a line each 10.7)
constexpr uint32_t kVerifyTickets = 1024, kVerifyTicketWords = 32;

// chunks of a prefix and a tail together
constexpr uint32_t kMaxParts = 1024;

// ---- prefix_attn: the prefix and each tail in chunks of keys, one workgroup
// each; a chunk's results (unnormalised sums, maximum and weight of the softmax)
// go to the workspace and are joined by a second launch.
// Few keys: one launch, a workgroup walks the prefix and its sequence's tail.  16-bit
// types up to 512 keys (MI355X, bf16, 32/8x128: 8 sequences of 5 tokens, 300 + 200
// keys, 9.9 us against 13.4 by chunks; 700 + 300 keys 13.8 against 10.8).  f32,
// whose products take eight times as long: where a sequence's pairs fill its tiles
// (64 sequences of 8 tokens, 300 + 200 keys: 47 against 68 us), and otherwise
// up to 128 keys, a subtile a wave, as the prefix shares its tiles between the
// sequences, and one launch is a longer chain for a few of them too (1 token,
// 32/8x128, 300 + 200 keys: 1 sequence 25.8 us against 16.4, 64 44.1 against 40.4;
// only near the limit one launch is ahead: 32/4x64, 128 + 64 keys, 2 sequences 9.2
// against 9.5, 64 9.7 against 13.0).
struct PrefixPlan {
    bool direct;
    uint32_t p_chunk, n_p;   // keys of a prefix chunk, chunks (0 without a prefix)
    uint32_t t_chunk, n_t;   // the same of a tail
    uint32_t p_slots;            // (query row, head of the group) pairs of a prefix tile
    uint32_t p_tiles, t_tiles;   // query tiles per KV head over the whole batch, and per sequence
    uint64_t rows;           // (query row, head) pairs
    uint64_t p_jobs, t_jobs;
    size_t ml_bytes, o_bytes;   // workspace: (m, l) pairs, then the sums

    size_t bytes() const { return ml_bytes + o_bytes; }
};

inline PrefixPlan prefix_plan(uint32_t prefix_len, uint32_t tail_cap, uint32_t n_seqs, uint32_t n_tokens,
                              uint32_t n_heads, uint32_t n_kv, uint32_t hd, uint32_t elem, uint32_t cus) {
    PrefixPlan p{};
    const uint64_t group = n_heads / n_kv, slots = (uint64_t)n_seqs * n_tokens * group;
    p.p_slots = elem == 2 && slots > kAttnTileRows ? 128u : kAttnTileRows;
    p.p_tiles = (uint32_t)((slots + p.p_slots - 1) / p.p_slots);
    p.t_tiles = (uint32_t)((n_tokens * group + kAttnTileRows - 1) / kAttnTileRows);
    // Enough chunks for two workgroups a CU, none below 256 keys (two subtiles of every wave; with 128, of one, 16-bit
    // types lose by the longer join, 12.9 -> 15.4 us for 13 sequences of 1 token behind 15001 rows, 17.0 -> 19.0 for 8 of
    // 5 behind 2048, and f32 gains where there are few sequences, 12.4 -> 10.4 for 2 behind 2048 + 256, and loses for 16
    // of 300 + 200 keys, 18.9 -> 19.9): the tails' fill up to
    // one a CU, the prefix' the rest, so that the two, which are bound by different things, run side by side (64
    // sequences of up to 1024 rows behind 32768, bf16: 87 us with two of the prefix a CU, 70 so; 16 of up to 300
    // behind 8192, f32: 46 and 36).
    auto split = [&](uint32_t keys, uint64_t per_chunk, uint64_t jobs, uint32_t *chunk, uint32_t *n) {
        if (!keys) return;
        uint64_t want = (jobs + per_chunk - 1) / per_chunk;
        const uint64_t most = (keys + 255) / 256;
        if (want > most) want = most;
        if (want > kMaxParts / 2) want = kMaxParts / 2;
        *chunk = (uint32_t)((((uint64_t)keys + want - 1) / want + 127) / 128 * 128);
        *n = (uint32_t)(((uint64_t)keys + *chunk - 1) / *chunk);
    };
    const uint64_t per_t = (uint64_t)p.t_tiles * n_kv * n_seqs;
    split(tail_cap, per_t, (prefix_len ? 1ull : 2ull) * cus, &p.t_chunk, &p.n_t);
    const uint64_t t_jobs = p.n_t * per_t;
    split(prefix_len, (uint64_t)p.p_tiles * n_kv, 2ull * cus - (t_jobs < cus ? t_jobs : cus), &p.p_chunk, &p.n_p);
    p.direct = (uint64_t)prefix_len + tail_cap <= (elem == 2 || n_tokens * group >= kAttnTileRows ? 512u : 128u);
    p.rows = (uint64_t)n_seqs * n_tokens * n_heads;
    p.p_jobs = (uint64_t)p.n_p * p.p_tiles * n_kv;
    p.t_jobs = (uint64_t)p.n_t * p.t_tiles * n_kv * n_seqs;
    const uint64_t parts = (uint64_t)(p.n_p + p.n_t) * p.rows;
    p.ml_bytes = (size_t)((parts * 8 + 255) / 256 * 256);
    p.o_bytes = (size_t)(parts * hd * 4);
    return p;
}

}  // namespace yule
