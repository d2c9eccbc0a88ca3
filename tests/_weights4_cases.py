"""Sizes at which the products with 4-bit weights take each of the library's kernels, by stk_4bit_product_kernel's numbers: with routing
(tokens, experts, top_k, inputs, outputs) and without (rows, inputs, outputs).  The inputs end inside a piece, and are more than a group of
any of GROUPS."""
GROUPS = [32, 64, 128, 256, 384]      # 256 and 384: several pieces with one scale
KERNELS = ["stream 8x1x1", "stream 4x1x2", "stream 4x1x4", "stream 2x2x2", "stream 1x4x4", "tile 32x128", "ring 32x256", "ring 32x128", "ring 16x128"]
ROUTED = {
    "stream 8x1x1": (20, 4, 2, 392, 80), "stream 4x1x2": (320, 2, 1, 392, 320), "stream 4x1x4": (320, 2, 1, 3080, 528), "stream 2x2x2": (320, 2, 1, 392, 800),
    "stream 1x4x4": (200, 64, 2, 392, 1040), "tile 32x128": (800, 8, 2, 395, 240), "ring 32x256": (800, 8, 2, 392, 2320), "ring 32x128": (800, 8, 2, 392, 528),
    "ring 16x128": (800, 8, 2, 392, 240),
}
PLAIN = {
    "stream 8x1x1": (3, 392, 80), "stream 4x1x2": (160, 392, 640), "stream 4x1x4": (160, 3080, 1120), "stream 2x2x2": (160, 392, 1600),
    "stream 1x4x4": (7, 392, 65552), "tile 32x128": (200, 395, 1904), "ring 32x256": (600, 392, 6672), "ring 32x128": (200, 392, 4624), "ring 16x128": (200, 392, 1904),
}
