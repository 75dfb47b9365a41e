"""Shapes of the batched operators' tests by the kernel that they are for: the
plan that they take is asserted on the CPU, and the GPU tests run them."""
from yule_amd import DType

BF16, F16, F32 = DType.BF16, DType.F16, DType.F32

# prompts that eight waves take, four of them every other tile of keys, by padded head size
# dtype, heads, KV heads, head_dim, lengths, slots, split
PROMPTS = [
    (dt, *shape, 128, 2)
    for dt in (F16, BF16)
    for shape in [(32, 8, 64, [1200]), (32, 4, 64, [1400]), (32, 4, 56, [1400]), (32, 8, 96, [1100])]
]

# heads, KV heads, head_dim, prefix, tail capacity, tail lengths, tokens; what the join's launch has: threads, lanes a chunk,
# loads ahead; by type: pairs of a prefix tile
PREFIXES = [
    # the join with loads ahead, for each number of lanes a chunk
    ((12, 2, 80, 15001, 100, [1 + 99 * s // 12 for s in range(13)], 1), (256, 32, 8), {F32: 32, F16: 128, BF16: 128}),
    ((4, 1, 64, 18100, 40, [40, 9], 1), (256, 16, 8), {F32: 32, F16: 32, BF16: 32}),
    ((8, 2, 256, 4000, 100, [100, 1, 0, 64, 33, 99, 2, 50], 2), (256, 64, 8), {F32: 32, F16: 128, BF16: 128}),
    # the join by one wave, and by four without loads ahead, over tiles that the prefix shares
    ((8, 2, 256, 700, 40, [40, 1, 0, 17, 33, 39, 2, 20], 2), (256, 64, 0), {F32: 32, F16: 128, BF16: 128}),
    ((8, 2, 64, 1500, 24, [24, 3, 0, 8, 24, 11, 1, 2, 24, 5], 2), (64, 16, 0), {F32: 32, F16: 128, BF16: 128}),
    ((16, 16, 256, 500, 70, [70 - s % 70 for s in range(64)], 64), (64, 64, 0), {F32: 32, F16: 128, BF16: 128}),
    # the same over tiles of few pairs; the other head sizes of f32
    ((4, 2, 64, 4000, 30, [30, 7], 1), (256, 16, 0), {F32: 32, F16: 32, BF16: 32}),
    ((6, 2, 80, 700, 70, [70, 5], 1), (64, 32, 0), {F32: 32, F16: 32, BF16: 32}),
    ((2, 1, 152, 600, 20, [20, 7], 1), (256, 64, 0), {F32: 32, F16: 32, BF16: 32}),
    ((2, 1, 168, 600, 20, [3, 20], 1), (256, 64, 0), {F32: 32, F16: 32, BF16: 32}),
    ((2, 1, 200, 600, 20, [20, 11], 1), (256, 64, 0), {F32: 32, F16: 32, BF16: 32}),
]

# in one launch, the head sizes of f32
SHORT = [(2, 1, hd, 60, 20, [20, 7], 2) for hd in (32, 80, 128, 168, 200, 256)]
