"""Shapes of products on 8-bit floats and the kernel that csrc/fp8_plan.h is to
send each to: side of the tiles (16: the kernel without tiles in LDS, by rows a
block), and whether none, all or some of the tiles are divided over the
contraction.  Shared by the CPU test that asks the plan and the GPU tests that
count on it."""

WHOLE, DIVIDED, PARTLY = "whole", "divided", "partly divided"

# (rows, n, k): (side, division), cut short on every side
TILES = {
    (70, 5737, 1040): (64, WHOLE),
    (40, 4103, 4112): (64, DIVIDED),
    (130, 5452, 3088): (64, PARTLY),
    (258, 7000, 784): (128, WHOLE),
    (70, 4103, 4112): (128, DIVIDED),
    (1030, 4103, 784): (128, PARTLY),
    (3000, 4103, 528): (256, WHOLE),
    (3337, 4740, 528): (256, PARTLY),
}
# whole tiles over many blocks of the contraction
DEEP = {
    (258, 5452, 6144): (64, WHOLE),
    (600, 4103, 6144): (128, WHOLE),
    (2040, 1400, 32768): (128, WHOLE),
    (3337, 4103, 6144): (256, WHOLE),
}
# without tiles: rows a block, or x brought over by the block itself
FEW = {
    (3, 300, 1040): (16, "own"),
    (17, 100, 2064): (16, 16),
    (17, 4103, 272): (16, 32),
    (40, 3000, 528): (16, 64),
}
