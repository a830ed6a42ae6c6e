"""Sizes that put the feed-forward products on each of their kernels: (rows, n, k) for every product, operand type and way
to run it.  Ragged in every direction: rows, columns and steps of the contraction end inside tiles."""

# product -> operands and output -> launches (kernel, "/parts" where the contraction is split) -> sizes
ROUTES = {
    ("linear", "half"): {
        "stream": (13, 88, 1160), "small": (45, 40, 168), "deep": (18828, 72, 176), "pair": (32953, 88, 168),
        "tall": (35178, 72, 240), "wide": (35645, 136, 168), "wide+small": (22231, 648, 168),
        "wide+deep": (4743, 3880, 272), "wide+pair": (10825, 3800, 240), "wide+tall": (2242, 8376, 784),
        "wide+wide": (2790, 8440, 6480)},
    ("linear", "e4m3"): {
        "stream": (13, 88, 1168), "small": (45, 40, 176), "deep": (18496, 72, 176), "pair": (37420, 72, 176),
        "tall": (34851, 72, 432), "wide": (34072, 136, 176), "wide+small": (2990, 5504, 176),
        "wide+deep": (12757, 1304, 528), "wide+pair": (17531, 3288, 288), "wide+tall": (6966, 5328, 848)},
    ("linear", "e4m3 to f32"): {
        "stream": (13, 88, 1168), "small": (45, 40, 176), "deep": (17799, 72, 176), "pair": (37386, 72, 176)},
    ("gated", "half"): {
        "stream": (13, 88, 1160), "small": (45, 40, 208), "deep": (129, 5952, 168), "pair": (36886, 40, 176),
        "tall": (36787, 40, 208), "wide": (35089, 72, 168), "wide+small": (8305, 984, 168),
        "wide+deep": (1212, 6560, 272), "wide+pair": (6503, 1896, 432), "wide+tall": (984, 8208, 880),
        "wide+wide": (1686, 6600, 5232)},
    ("gated", "e4m3"): {
        "stream": (13, 88, 1168), "small": (45, 40, 176), "deep": (74, 8632, 176), "pair": (34569, 40, 176),
        "tall": (33952, 40, 480), "wide": (36218, 72, 176), "wide+small": (1362, 5960, 176),
        "wide+deep": (2579, 3320, 416), "wide+pair": (4384, 4600, 432), "wide+tall": (11654, 1664, 784),
        "wide+wide": (1240, 8520, 5600)},
    ("dx", "half"): {
        "small": (44, 152, 48), "small/parts": (40, 1080, 56), "deep": (17573, 200, 80), "deep/parts": (65, 3432, 3056),
        "pair": (34480, 168, 56), "pair/parts": (67, 2520, 5856), "wide": (32894, 168, 168),
        "wide/parts": (141, 8872, 2944), "wide+small": (17041, 152, 976), "wide+deep": (20115, 392, 800),
        "wide+pair": (2699, 424, 7552), "wide+wide": (2710, 5512, 8288)},
    ("dw", "half"): {
        "small": (151, 40, 48), "small/parts": (979, 40, 48), "deep": (151, 264, 6544), "deep/parts": (7176, 72, 1360),
        "pair": (154, 8816, 400), "pair/parts": (4035, 2752, 80), "wide": (161, 5992, 1344),
        "wide/parts": (6061, 136, 5680), "wide+small": (153, 2088, 8176), "wide+deep": (464, 6088, 2832),
        "wide+pair": (530, 2864, 7280), "wide+wide": (8843, 5552, 7344)},
}


def route(launches):
    """"kernel", "kernel/parts" or "kernel+kernel" of hip.linear_plan's answer."""
    return "+".join(kernel + ("/parts" if parts > 1 else "") for kernel, parts, _ in launches)
