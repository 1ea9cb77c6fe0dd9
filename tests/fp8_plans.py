"""Sizes (rows, matrix rows, columns) that bring every kernel of the products in 8-bit floating point, with one part of the columns and with several, matrices whose rows end on 16 bytes of output and whose do not:
{sizes: (plan of 32-bit outputs, plan of 16-bit outputs)}, a plan being (matrix rows of a tile, rows of a tile, parts), (0, 0, 1) the stream.  And what the sums of a product are off by."""
import ctypes as C

import inferflow_amd as ia

PLANS = {
    (1, 130, 400): ((0, 0, 1), (0, 0, 1)), (16, 4096, 2064): ((0, 0, 1), (0, 0, 1)), (18, 59, 64): ((0, 0, 1), (0, 0, 1)), (19, 48, 64): ((0, 0, 1), (0, 0, 1)),
    (19, 48, 5136): ((128, 32, 14), (128, 32, 14)), (23, 50, 5136): ((128, 32, 14), (128, 32, 14)), (24, 11008, 4096): ((128, 32, 5), (128, 32, 5)), (40, 4096, 4096): ((128, 32, 4), (128, 32, 8)),
    (64, 4096, 11008): ((128, 64, 8), (128, 64, 8)), (128, 4096, 4096): ((128, 64, 4), (128, 64, 4)), (256, 4096, 4096): ((128, 64, 2), (128, 64, 2)), (512, 4096, 4096): ((128, 64, 1), (128, 64, 1)),
    (1024, 4096, 4096): ((128, 128, 1), (128, 64, 1)), (516, 13120, 80): ((128, 64, 1), (256, 256, 1)), (3647, 648, 13904): ((256, 128, 2), (256, 256, 5)), (3666, 1064, 1536): ((256, 128, 1), (256, 128, 1)),
    (3716, 56, 4096): ((128, 64, 4), (128, 64, 4)), (3742, 49, 3648): ((0, 0, 1), (128, 64, 4)), (3819, 1048, 688): ((256, 128, 1), (128, 128, 1)), (3902, 645, 14416): ((256, 128, 2), (256, 256, 5)),
    (4039, 104, 1040): ((128, 32, 1), (128, 32, 1)), (4085, 50, 4048): ((128, 64, 4), (128, 64, 4)), (4097, 137, 8080): ((256, 128, 7), (128, 128, 7)), (4098, 130, 976): ((0, 0, 1), (128, 64, 1)),
    (4099, 48, 15872): ((128, 128, 7), (128, 128, 14)), (4102, 144, 1280): ((128, 64, 1), (128, 64, 1)), (4127, 56, 3984): ((128, 128, 7), (128, 64, 7)), (4147, 136, 6256): ((256, 128, 7), (128, 64, 3)),
    (4171, 934, 688): ((256, 128, 1), (128, 128, 1)), (4179, 133, 9104): ((256, 128, 7), (256, 128, 6)), (4229, 49, 3504): ((128, 128, 7), (128, 64, 7)), (4262, 408, 928): ((128, 128, 1), (128, 64, 1)),
    (4326, 389, 1008): ((128, 128, 1), (128, 64, 1)), (4370, 144, 9072): ((256, 128, 7), (256, 128, 6)), (4561, 129, 960): ((128, 64, 1), (128, 64, 1)), (4642, 1683, 144): ((128, 64, 1), (256, 256, 1)),
    (4666, 82, 1040): ((0, 0, 1), (128, 32, 1)), (4681, 89, 1056): ((128, 32, 1), (128, 32, 1)), (4686, 800, 112): ((128, 64, 1), (128, 128, 1)), (4698, 815, 1296): ((256, 128, 1), (256, 128, 1)),
    (4701, 794, 176): ((128, 64, 1), (128, 128, 1)),
}


def plan(tokens, rows, cols, dtype, ws_bytes=None, lda=None):
    tile = [C.c_int(-7) for _ in range(3)]
    if ws_bytes is None:
        ws_bytes = ia.lib().ifa_linear_fp8_workspace_bytes(rows, cols, tokens)
    ia.check(ia.lib().ifa_linear_fp8_plan(rows, cols, cols if lda is None else lda, tokens, dtype, ws_bytes, *(C.byref(v) for v in tile)))
    return tuple(v.value for v in tile)


def limit_32(blocks):
    """What all values of a 32-bit product together are off by, against their size: a block's sum (of exact products; the matrix cores' 32-bit sums, two roundings in all as measured with pairs of blocks) is
    scaled and added to those before, over at most 16 waves or parts; each of these roundings is off by 2^-24 of the sum at most, and no two alike."""
    return (2 + (35 + blocks) ** 0.5) * 2.0 ** -24
