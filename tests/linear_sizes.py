"""Products long enough for the steady state of their kernels, and which kernel each is: test_language_layers_cpu.py checks that it is launched, test_gpu_linear_plan.py its results.

A wavefront of linear_rows_kernel takes every eighth block of k and has two under way: its loop without conditions needs 32 blocks, with 37, 51 and 69 some wavefronts
have one more than others.  linear_tile_kernel has a ring of three blocks: from the fourth on a place is written again."""
HALF, INT8, FLOAT = 0, 1, 2  # float16 rows and weights; int8 weights; float32
BLOCK = {HALF: 64, INT8: 64, FLOAT: 32}  # k of a block

# kernel: ("rows", tiles of 16 rows, fragments of 16 columns) or ("tile", rows);  type, kernel, rows, blocks of k, columns
PLAIN = [
    (HALF, ("rows", 1, 1), 1, 69, 200), (HALF, ("rows", 1, 4), 8, 37, 9000), (HALF, ("rows", 2, 1), 9, 37, 400), (HALF, ("rows", 2, 1), 31, 69, 1000), (HALF, ("rows", 2, 2), 64, 32, 2100),
    (HALF, ("rows", 2, 4), 17, 51, 10000), (HALF, ("rows", 2, 4), 128, 37, 2100), (HALF, ("rows", 4, 4), 64, 51, 8300), (HALF, ("rows", 4, 4), 200, 33, 4000),
    (HALF, ("tile", 64), 300, 4, 5000), (HALF, ("tile", 64), 500, 7, 3500), (HALF, ("tile", 128), 1000, 4, 4090), (HALF, ("tile", 128), 1300, 11, 2800),
    (HALF, ("tile", 256), 2000, 4, 4300), (HALF, ("tile", 256), 2049, 5, 4300), (HALF, ("tile", 256), 1800, 13, 5000),
    (INT8, ("rows", 1, 2), 7, 51, 300), (INT8, ("rows", 2, 2), 9, 32, 500), (INT8, ("rows", 2, 2), 60, 69, 2000), (INT8, ("rows", 2, 4), 33, 37, 4500), (INT8, ("rows", 4, 4), 50, 51, 9000),
    (INT8, ("rows", 4, 4), 300, 37, 5000), (INT8, ("tile", 64), 300, 5, 11500), (INT8, ("tile", 128), 1000, 7, 4090), (INT8, ("tile", 256), 2000, 4, 4300), (INT8, ("tile", 256), 1500, 9, 6000),
    (FLOAT, ("rows", 1, 1), 5, 69, 100), (FLOAT, ("rows", 2, 1), 20, 37, 900), (FLOAT, ("rows", 2, 2), 64, 51, 2100), (FLOAT, ("rows", 2, 4), 100, 32, 2100), (FLOAT, ("rows", 4, 4), 512, 37, 2000),
    (FLOAT, ("rows", 4, 2), 64, 33, 17000), (FLOAT, ("tile", 64), 700, 4, 2900), (FLOAT, ("tile", 64), 1000, 11, 4000),
]

# the same over experts: type, kernel, experts, rows of x to a row of the result, rows, blocks of k, columns
EXPERTS = [
    (HALF, ("rows", 1, 4), 64, 8, 128, 37, 256), (HALF, ("rows", 2, 1), 3, 1, 40, 51, 60), (HALF, ("rows", 2, 2), 8, 1, 100, 33, 750), (HALF, ("rows", 2, 4), 20, 2, 300, 69, 900),
    (HALF, ("tile", 64), 10, 2, 700, 5, 300), (HALF, ("tile", 128), 5, 1, 1000, 7, 500), (HALF, ("tile", 256), 3, 3, 1200, 4, 700), (HALF, ("tile", 256), 7, 1, 4000, 9, 300),
    (INT8, ("rows", 1, 4), 64, 8, 128, 37, 300), (INT8, ("rows", 2, 2), 3, 1, 30, 51, 200), (INT8, ("rows", 2, 4), 30, 1, 300, 37, 700), (INT8, ("tile", 64), 20, 4, 1000, 5, 200),
    (INT8, ("tile", 128), 4, 1, 1500, 11, 500), (FLOAT, ("rows", 1, 1), 2, 1, 14, 37, 70), (FLOAT, ("rows", 2, 4), 20, 2, 400, 32, 800), (FLOAT, ("rows", 2, 2), 8, 1, 96, 51, 750),
    (FLOAT, ("tile", 64), 6, 1, 900, 7, 300),
]
