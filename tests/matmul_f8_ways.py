"""Sizes of products of operands in 8 bits at which each way of computing one is chosen (on 256 compute
units): (fp32 result, m, n, k, way of f8_routes.h). test_f8_routes.py holds the choice to them on the CPU,
test_matmul_f8_tiles_gpu.py runs them. The ways of tiles of 128 rows and more are there with more tiles than compute units,
so that workgroups take several, ragged in both directions, and with K of as few slices as choose them."""

SPLIT, STREAM_16X64, STREAM_32X32, STREAM_32X64, STREAM_64X64, TILES_128, TILES_128X256, TILES_256 = range(8)

WAYS = [
    (0, 5, 1000, 700, SPLIT),
    (0, 16, 9001, 2001, STREAM_16X64),
    (0, 60, 2001, 4000, STREAM_32X32),
    (0, 130, 3001, 900, STREAM_32X64),
    (0, 400, 2999, 700, STREAM_64X64),
    (0, 4101, 4507, 100, TILES_128),
    (0, 1501, 6803, 200, TILES_128),
    (0, 1101, 5505, 300, TILES_128),
    (0, 2300, 4300, 640, TILES_128),
    (0, 4501, 6305, 100, TILES_128X256),
    (0, 4900, 2707, 200, TILES_128X256),
    (0, 4100, 4300, 640, TILES_128X256),
    (0, 1701, 5003, 1000, TILES_128X256),
    (0, 20001, 11003, 100, TILES_256),
    (0, 10301, 9002, 300, TILES_256),
    (0, 5000, 5000, 1024, TILES_256),
    (0, 4401, 5402, 1500, TILES_256),
    (1, 5, 1000, 700, SPLIT),
    (1, 16, 9001, 2001, STREAM_16X64),
    (1, 60, 2001, 4000, STREAM_32X32),
    (1, 130, 3001, 900, STREAM_32X64),
    (1, 400, 2999, 700, STREAM_64X64),
    (1, 5000, 3101, 640, TILES_128),
    (1, 5501, 1300, 1500, TILES_128),
    (1, 3803, 5702, 100, TILES_128X256),
    (1, 3101, 4305, 200, TILES_128X256),
    (1, 4100, 4300, 640, TILES_128X256),
    (1, 1501, 6803, 1000, TILES_128X256),
]
