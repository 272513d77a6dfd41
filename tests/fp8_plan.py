"""Which form an e4m3 product takes, and in how many parts along K: the library's rule on the host again, with the constants of its source,
so that tests can say which forms their sizes reach."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "webdnn_amd", "csrc", "gemm_fp8.hip")


def _constants():
    text = open(SOURCE).read()
    table = re.search(r"constexpr Form forms\[FORMS\] = \{(.*?)\};", text, re.S).group(1)
    forms = [[float(x.rstrip("f")) for x in row.split(",")] for row in re.findall(r"\{([^{}]*)\}", table)]
    return [(int(c), int(r), start, block) for c, r, start, block in forms], int(re.search(r"FIRST_TILES = (\d+)", text).group(1))


FORMS, FIRST_TILES = _constants()


def plan(m, n, k, cus=256):
    """(form, parts): "rows" for one or two rows, else an index of FORMS."""
    if m <= 2:
        return "rows%d" % m, 1
    aligned, blocks = k % 16 == 0, -(-k // 128)
    best, least = None, None
    for form, (cols, rows, start, block) in enumerate(FORMS):
        tiles, direct = -(-n // cols) * -(-m // rows), form < FIRST_TILES
        if direct and not aligned:
            block *= 1.4
        turns = 4 if form == FIRST_TILES - 1 else 8
        for cut in (False, True):
            parts = min(cus // tiles if cut else 1, blocks)
            if cut and parts < 2:
                continue
            part = -(-blocks // parts) if parts > 1 else blocks
            if parts > 1:
                parts = -(-blocks // part)
            us = -(-tiles * parts // cus) * (start + block * (-(-part // turns) * turns if direct else part))
            if parts > 1:
                us += 4 + parts * (0.15 + m * n * 8e-7)
            if not direct and not aligned:
                us += 3 + (m + n) * k * 4e-7
            if least is None or us < least:
                best, least = (form, parts), us
    return best


def kind(m, n, k):
    form, parts = plan(m, n, k)
    return form, k % 16 == 0, parts > 1


# A case of each form, with rows of whole 16-byte pieces and without, whole and cut along K.
CASES = [(1, 130, 2000), (1, 77, 4100), (2, 300, 2064), (2, 131, 1030),
         (3, 21, 2109), (5, 83, 6231), (7, 29, 3088), (4, 98, 9232),
         (19, 61, 1001), (69, 1, 6754), (9, 55, 1040), (34, 2, 11296),
         (395, 636, 129), (3, 1404, 6047), (387, 629, 144), (3, 1864, 6176),
         (341, 356, 130), (459, 1, 8541), (371, 321, 272), (401, 1, 9936),
         (550, 452, 131), (17, 1075, 7703), (501, 514, 144), (364, 70, 8176),
         (747, 647, 130), (2147, 1, 27659), (689, 756, 400), (4484, 1, 14432),
         (787, 1228, 300), (1384, 379, 3639), (674, 714, 144), (1364, 73, 9328),
         (1486, 1322, 200), (9467, 71, 3385), (1482, 1315, 144), (8491, 68, 2976),
         (2105, 1957, 150), (5825, 147, 3798), (1925, 2077, 272), (71, 11770, 3792)]
