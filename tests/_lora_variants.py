"""Calls of lora_add that between them take every way that its sizes choose among: for the GPU tests, and for a check
on the CPU that they do."""
import numpy as np

# sequences, rows (1: each has one, and no starts; -k: k each; k: up to k), adapters, max_rank, in_features, part_ends
SIZES = [
    # one launch: 256, 512 and 1024 columns a block, one and two products, a tile's blocks together and spread
    (1, 1, 4, 16, 2048, (2048,)), (1, 1, 4, 16, 512, (16384,)), (1, 1, 2, 32, 264, (40960,)), (5, 1, 3, 16, 264, (24576,)),
    (40, 1, 40, 16, 520, (2048,)), (40, 1, 40, 32, 520, (2048,)), (64, 3, 30, 24, 264, (1024, 2048)),
    (20, 9, 20, 16, 72, (8192,)), (12, 10, 12, 32, 72, (8192,)), (48, 5, 16, 16, 4096, (4096, 5120, 6144)),
    (50, 5, 16, 32, 1024, (4096, 5120)), (60, 6, 16, 32, 1024, (16384,)), (5, 1, 5, 16, 264, (49152,)),
    (5, 1, 5, 32, 264, (49152,)), (30, 4, 8, 32, 1024, (32768,)), (5, 1, 3, 32, 264, (24576,)), (200, 1, 12, 16, 136, (1024,)), (300, 1, 20, 24, 136, (512,)),
    # two: few tiles, whose products and in_features are shared out
    (1, 1, 2, 64, 8192, (1000,)), (3, 1, 2, 128, 4104, (11008, 22016)), (2, 5, 2, 16, 16392, (520,)), (1, 9, 1, 256, 8192, (264,)),
    (4, 1, 4, 128, 8192, (2048,)), (6, 1, 6, 72, 6152, (512, 1024)), (40, 1, 20, 48, 2056, (4096, 5120, 6144)),
    (32, 1, 4, 32, 8192, (4096, 5120, 6144)), (17, 1, 1, 128, 4096, (4096, 5120, 6144)), (2, 30, 2, 40, 1032, (64, 128, 200)),
    # and many, for which a block of the second launch takes some in a row
    (6, 600, 4, 32, 2048, (8192, 16384)), (5, 700, 3, 16, 136, (8192, 16384)), (256, 5, 30, 64, 8192, (16384,)),
    (200, 4, 12, 32, 8192, (40960,)), (130, 40, 7, 64, 264, (8192,)), (3, 456, 3, 128, 8192, (11008, 22016)),
    (4, 500, 2, 256, 1024, (8192,)), (70, 8, 5, 128, 8192, (16384,)), (60, 1, 8, 128, 8192, (16384,)),
    (300, 2, 3, 16, 4096, (16384,)), (600, 3, 9, 48, 72, (4096, 8192)), (24, 80, 1, 32, 520, (16384,)),
    (40, 40, 40, 256, 2048, (4096,)), (9, 200, 5, 96, 264, (4096, 8192, 12288)), (700, 1, 300, 32, 520, (2048, 4096)), (20, 3, 2, 256, 136, (520,)),
    (300, 20, 3, 16, 8192, (16384,)), (90, 1, 8, 128, 8192, (40960,)), (150, 12, 6, 16, 1032, (2048, 2568, 3200)),
    (400, 1, 120, 16, 1032, (2048, 2568, 3200))]


class Sizes:
    def __init__(self, at):
        self.n, rows, self.adapters, self.rank, self.inner, self.ends = SIZES[at]
        self.rng = np.random.default_rng([at, self.n, self.rank])
        self.rows = None if rows == 1 else self.rng.integers(1, rows + 1, self.n)
        if self.rows is not None:
            self.rows[0] = rows
        self.n_rows = self.n if self.rows is None else int(self.rows.sum())

    def call(self):
        return self.n_rows, self.n, self.adapters, self.rank, self.inner, self.ends
