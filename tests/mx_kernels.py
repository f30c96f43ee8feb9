"""Which kernel a product of MX rows takes, as ns_mx_linear.h chooses it, and sizes that take each of them."""

UNITS, FULL = 256, 200


def kernel_of(fmt, m, n, k):
    """The template arguments after the result's type: ("few", format, U, KS) or ("tile", format, BM, BN, WM, WN, BK, P, SP)."""
    tiles = lambda bm, bn: -(-m // bm) * -(-n // bn)  # noqa: E731
    few = lambda f: ("few", f, *((2, 16) if k <= 2048 else (4, 64)))  # noqa: E731
    if fmt == "mxfp8":
        if m <= 16 and n <= 2 * 32 * UNITS:
            return few(8)
        if m > 64 and tiles(128, 256) >= FULL:
            return ("tile", 8, 128, 256, 2, 2, 128, 2, 4)
        if tiles(64, 32) <= UNITS:
            return ("tile", 8, 64, 32, 4, 1, 256, 4, 4)
        if tiles(64, 64) <= 2 * UNITS:
            return ("tile", 8, 64, 64, 4, 1, 256, 2, 2)
        return ("tile", 8, 64, 128, 2, 2, 256, 2, 2)
    if m <= 16 and n <= 32 * UNITS:
        return few(4)
    if m > 128 and tiles(128, 128) > 2 * UNITS:
        return ("tile", 4, 256, 256, 4, 2, 256, 2, 2)
    if m > 64 and tiles(64, 128) > UNITS:
        return ("tile", 4, 128, 128, 2, 2, 256, 2, 2)
    if tiles(64, 128) >= 2 * UNITS:
        return ("tile", 4, 64, 128, 2, 2, 256, 2, 2)
    if FULL <= tiles(64, 128) <= UNITS:
        return ("tile", 4, 64, 128, 2, 2, 256, 3, 4)
    return ("tile", 4, 64, 64, 2, 2, 256, 4, 4)


def round_of(kernel):
    """Columns after which a kernel's loop begins again: a round of the waves' groups, or the unrolled stages."""
    if kernel[0] == "few":
        return 128 * kernel[3]
    bk, p, sp = kernel[6:]
    stages = p
    while stages % (2 * sp):
        stages += p
    return stages * bk


def widths(kernel):
    """Padded widths of one stage, of less than a round, one, and past it by a whole stage, a part of one and another round."""
    r = round_of(kernel)
    if kernel[0] == "few" and kernel[2] == 2:
        return [128, 256, 384, 1920, 2048]
    first = [2176] if kernel[0] == "few" else [128, 256, 384]
    return first + [r - 128, r, r + 128, 2 * r + 384]


# (format, rows, outputs): ragged on both sides, every wave's part of a tile in use somewhere
SIZES = [("mxfp8", m, n) for m, n in
         ((1, 33), (16, 97), (5, 16384),                       # few rows
          (17, 40), (64, 8192), (200, 2000),                   # 64 x 32
          (64, 8200), (300, 6500),                             # 64 x 64
          (64, 32832), (330, 5700), (16, 32900),               # 64 x 128
          (65, 51250), (300, 17000), (2600, 2400))] + [        # 128 x 256
         ("mxfp4", m, n) for m, n in
         ((1, 33), (16, 97), (5, 8192),                        # few rows
          (17, 70), (64, 12000), (300, 3000), (50, 40000),     # 64 x 64
          (64, 25700), (129, 8600),                            # 64 x 128, three places
          (64, 65600), (33, 65700),                            # 64 x 128, two places
          (140, 12900), (700, 4300),                           # 128 x 128
          (300, 25700), (2700, 4700))]                         # 256 x 256


def kernels_of(fmt, m, n):
    """The kernels that a size takes over all widths."""
    return [kernel_of(fmt, m, n, 128)] + ([kernel_of(fmt, m, n, 4096)] if kernel_of(fmt, m, n, 128)[0] == "few" else [])
