"""Calls of linear by the form that each takes (not collected by pytest): (form, whether each CU has one tile at most, MX, rows,
inputs, matrix rows), matrix rows being the outputs, with SwiGLU twice as many.  Every form of either format, and both instances
of those that differ where no CU has two tiles; odd rows, outputs off the tiles, inputs off a step where the form takes any,
enough of them for every stage to be filled twice."""
FORMS = [
    ("few", False, False, 1, 1000, 514), ("few", False, False, 2, 136, 34), ("few", False, False, 3, 72, 10),
    ("few", False, False, 4, 2560, 642),
    ("16", True, False, 17, 1096, 18), ("16", False, False, 17, 1096, 2058),
    ("32", True, False, 33, 584, 2744), ("32", False, False, 4109, 584, 66),
    ("32x64", True, False, 2755, 328, 66), ("64", False, False, 5529, 328, 132), ("64deep", True, False, 5453, 648, 66),
    ("64deep", True, False, 2047, 2048, 510),
    ("128", True, False, 5549, 176, 130), ("128", False, False, 6671, 176, 518),
    ("128x320", True, False, 6571, 496, 1158), ("256", True, False, 5895, 168, 1314), ("256x320", True, False, 6473, 168, 2312),
    ("few", False, True, 1, 1056, 514), ("few", False, True, 2, 160, 34), ("few", False, True, 3, 96, 10),
    ("few", False, True, 4, 2560, 642),
    ("16", True, True, 17, 2208, 18), ("16", False, True, 17, 2208, 2058),
    ("32", True, True, 33, 1184, 2724), ("32", False, True, 4111, 1280, 34),
    ("32x64", True, True, 2743, 608, 66), ("64", False, True, 6151, 640, 194),
    ("128", True, True, 6697, 384, 260), ("128", False, True, 6557, 384, 516),
    ("128x320", True, True, 7219, 384, 1032),
]
