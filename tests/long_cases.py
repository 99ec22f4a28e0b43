"""Attention calls whose tensor-core prefix items are long: every ring slot of the prefix kernel is reused many times.
test_batch_host.py holds the cut to that, test_gpu_long_prefix.py runs them."""

# Tiles that an item has at least.  The kernel's rings have at most 16 slots and an item two ring items a tile, so each
# slot is used five times or more (and each staging slot of a coded prefix's warps several times).
LEAST_TILES = 40

# hq, hkv, dim, batch, prefix, page, dtype; page 0: coded.  Pages of 16, 24, 64 and 128 tokens come by TMA, of 7 and 20 by rows.
CASES = [
    (37, 37, 32, 21, 21003, 0, "bf16"), (74, 37, 64, 70, 11111, 0, "bf16"), (148, 148, 128, 30, 2800, 0, "bf16"),
    (37, 37, 256, 9, 11008, 0, "bf16"), (32, 8, 128, 33, 47003, 0, "bf16"), (8, 8, 256, 130, 47003, 0, "bf16"),
    (74, 74, 32, 40, 11007, 7, "bf16"), (74, 74, 32, 33, 11007, 20, "fp16"), (74, 74, 64, 12, 11007, 20, "bf16"),
    (148, 74, 64, 70, 11007, 7, "fp16"), (74, 74, 128, 17, 11007, 7, "bf16"), (74, 74, 128, 40, 11007, 20, "fp16"),
    (74, 74, 256, 10, 5600, 20, "bf16"), (37, 37, 256, 33, 11007, 7, "fp16"),
    (74, 74, 32, 33, 11007, 16, "bf16"), (74, 74, 64, 33, 11007, 24, "fp16"), (74, 74, 128, 20, 11007, 64, "bf16"),
    (37, 37, 256, 20, 11007, 128, "fp16"),
]
