"""Sizes that reach every form of the token-head kernels: the tiles of the linear layer's products and the ways in which a row of the norms is
held.  test_token_forms.py asks the library which form each size takes; test_gpu_token_forms.py runs them."""

# rows, width, out, activation, bias, residual; what the 16-bit types take: (forward, dx) tiles, whether rows begin at 16 bytes
LINEAR = [
    (8200, 1000, 1032, "gelu", True, True, (128, 128), True),       # remainders of rows, columns and steps, sixteen steps
    (8199, 1001, 1030, "silu", True, True, (128, 128), False),
    (12300, 1160, 1160, "relu", True, True, (256, 256), True),
    (12300, 1160, 1160, "gelu", True, False, (256, 256), True),
    (16389, 136, 1288, "silu", False, True, (256, 64), True),       # a short contraction forward, a long one back
    (16389, 1288, 136, "none", True, True, (64, 256), True),
    (16389, 1287, 135, "none", True, False, (64, 128), False),
    (40003, 128, 128, "relu", True, False, (128, 128), True),       # the towers' own width
    (40003, 128, 128, "silu", False, True, (128, 128), True),
    (30001, 129, 131, "relu", False, False, (128, 128), False),
    (8200, 1000, 1032, "none", False, False, (128, 128), True),
    (300, 2000, 2000, "gelu", True, True, (64, 64), True),
    (301, 1999, 2001, "relu", True, True, (64, 64), False),
]

# f32 products of few tiles, whose contraction is split over workgroups: rows, width, out, activation, bias, residual; whether the forward and dx split
SPLIT = [
    (60, 2560, 2560, "gelu", True, True, (True, True)),
    (1, 2560, 130, "silu", True, False, (True, False)),
    (37, 2369, 1281, "relu", True, True, (True, True)),             # rows at no multiple of 16 bytes, remainders everywhere
    (1040, 2560, 320, "relu", True, False, (True, False)),
    (1108, 2562, 639, "none", True, True, (True, False)),
    (260, 72, 2560, "silu", False, True, (False, True)),
    (3, 33, 5000, "gelu", True, False, (False, True)),
    (8926, 1617, 80, "silu", True, False, (True, False)),
    (4096, 2560, 640, "gelu", True, True, (True, False)),
]

# batch, tokens, width, gate, after, before, kind, residual, scale: aligned rows of every width that is held another way
NORM = [
    (3, 50, 16, "element", "affine", "affine", "layer", True, 0.5), (3, 50, 64, "sequence", "affine", "affine", "rms", True, 0.5),
    (3, 50, 72, "keep", "affine", "affine", "layer", True, 1 / 0.9), (3, 50, 192, "sequence", "affine", "affine", "layer", True, 0.5),
    (3, 50, 256, "keep", "affine", None, "layer", False, 1 / 0.9), (4, 60, 320, "element", "affine", "affine", "rms", True, 0.25),
    (2, 80, 512, "channel", None, "affine", "layer", True, 1.0), (3, 70, 768, "keep", "affine", "affine", "layer", True, 1 / 0.9),
    (2, 90, 520, "sequence", "affine", "plain", "rms", True, 0.5), (3, 50, 896, "element", "affine", "affine", "layer", True, 0.5),
    (5, 40, 1024, "sequence", "plain", "affine", "layer", True, 0.5), (3, 50, 1280, "channel", "affine", "affine", "rms", True, 0.25),
    (2, 60, 2048, "keep", "affine", "affine", "layer", True, 1 / 0.9), (3, 30, 2560, "sequence", "affine", "affine", "layer", True, 0.5),
    (2, 30, 4096, "element", "affine", "affine", "rms", True, 0.5), (700, 3, 1280, "sequence", "affine", "affine", "layer", True, 0.5),
    (3, 50, 1282, "element", "affine", "affine", "layer", True, 0.5), (3, 50, 700, "sequence", "affine", "affine", "layer", True, 0.5),
    (3, 50, 701, "channel", "affine", "affine", "layer", True, 0.5), (2, 50, 2052, "keep", "plain", "affine", "layer", True, 0.5),
    (2, 50, 3001, "channel", "affine", "affine", "layer", True, 0.5), (2, 50, 901, "sequence", "affine", "affine", "rms", True, 0.5),
    (2, 50, 203, "element", "affine", "affine", "rms", True, 0.5), (2, 50, 405, "keep", "affine", "affine", "layer", True, 0.5),
    (2, 50, 33, "keep", "affine", "affine", "layer", True, 0.5), (2, 50, 101, "element", "affine", "affine", "layer", True, 0.5),
    (2, 50, 1501, "element", "affine", "affine", "layer", True, 0.5),
]
