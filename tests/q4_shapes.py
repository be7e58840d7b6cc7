"""Sizes of products with 4-bit weights that between them take every kernel, tile and way of cutting that the plan has on 148 SMs."""

SMS = 148
# (tokens, rows, rows of a gated product, values of a row): odd ends of the last tile of rows, the last block and the last group of k in most of them
SHAPES = [(5, 100, 128, 136), (5, 9000, 9088, 136), (8, 1000, 1024, 1032), (13, 100, 128, 136), (13, 9000, 9088, 136), (16, 333, 384, 3080),
          (20, 333, 384, 1032), (31, 9000, 9088, 136), (32, 1000, 1024, 4104), (40, 333, 384, 1032), (63, 9000, 9088, 264), (64, 1000, 1024, 4104),
          (66, 100, 128, 3080), (96, 1000, 1024, 4096), (97, 1000, 1024, 4104), (100, 2000, 2048, 4104), (128, 3500, 3584, 4104), (256, 3500, 3584, 4104),
          (300, 5000, 5120, 8200), (66, 100, 128, 136), (97, 5000, 5120, 520), (129, 9590, 9600, 136), (200, 5000, 5120, 520), (161, 19000, 19072, 264),
          (300, 5000, 5120, 136), (700, 9000, 9088, 520), (100, 38000, 38016, 264), (700, 3500, 3584, 3080), (500, 5000, 5120, 8200), (400, 5000, 5120, 4104)]


def ways(plan, n, sms=SMS):
    """What a plan's launches have of their own: (kernel, tokens of a tile, more than one range of K; for persistent blocks more than one tile each)."""
    return {(kernel, tile, -(-n // 128) * -(-tokens // tile) > sms if kernel == "gemm_q4_long" else ranges > 1) for tokens, kernel, tile, ranges in plan}
