"""Calls of the head's loss by how the products are tiled and split: (tokens, width, vocabulary, piece or None) and, for
the logits, dx and dw, the tile's columns and which tiles are split over K ("whole": none, "tail": those of the last
round, "all").  The sizes are odd in every direction; where there are pieces, the last one is shorter."""

HEAD_PATHS = [
    ((74, 808, 332, None), "128 all, 128 whole, 256 whole"),
    ((206, 3416, 5370, None), "128 all, 128 all, 256 whole"),
    ((147, 3408, 33073, None), "128 tail, 256 all, 256 whole"),
    ((940, 840, 17143, None), "256 tail, 128 all, 256 tail"),
    ((3278, 3624, 1161, None), "256 all, 256 whole, 256 all"),
    ((7319, 2136, 517, None), "128 whole, 256 tail, 256 all"),
    ((10927, 528, 1575, None), "256 whole, 128 tail, 256 all"),
    ((79, 744, 325, 65), "128 all, 128 whole, 256 whole"),
    ((297, 2616, 32919, 180), "128 tail, 256 all, 256 whole"),
    ((1129, 784, 22403, 645), "256 tail, 128 all, 256 whole"),
    ((860, 272, 33301, 695), "256 whole, 128 all, 256 tail"),
    ((6881, 1384, 1577, 5386), "256 whole, 128 tail, 256 all"),
    ((12296, 1400, 577, 10885), "256 whole, 256 tail, 256 all"),
]
