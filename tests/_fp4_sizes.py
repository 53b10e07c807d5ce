"""Sizes of the FP4 linear layers that between them take every form of the kernels for five rows and more over a K of
eight slabs of 64 columns and more for each wave, so that every place of its rings is refilled, with a last slab of 32
columns. (rows, in, out), for SwiGLU (rows, hidden, inter)."""

LINEAR_LONG = [(9, 3168, 40), (1400, 992, 167), (1381, 2336, 40), (1433, 3104, 40), (1403, 1056, 264), (1441, 1696, 99),
               (1392, 4128, 65), (1367, 928, 645), (1442, 1952, 164), (1477, 800, 391), (1439, 544, 359), (612, 480, 3301),
               (500, 544, 4608), (1350, 672, 1428), (1347, 1440, 2216), (700, 3616, 4608), (1415, 1824, 2696),
               (1441, 1952, 2998)]

SWIGLU_LONG = [(1364, 864, 96), (1322, 2144, 32), (10, 3104, 32), (1366, 1056, 144), (1464, 1568, 64), (1378, 3872, 48),
               (1406, 928, 336), (1416, 1824, 96), (1191, 800, 256), (1292, 544, 208), (231, 480, 4336), (1431, 544, 720),
               (1351, 1440, 1152), (1425, 1568, 1376), (1350, 1056, 1808)]
