"""Which kernels one routed_experts call launches: the host rules of cfmoe_routed_experts,
written again, with the column tiles that its runs of pairs take.

A kernel is named by its template's values as the compiler spells them, so that the
names can be compared with those in the built library.
"""

from __future__ import annotations

UP_BF16, UP_FP4, DOWN_FP4 = range(3)
EXACT, RAGGED, HALF_STEP = range(3)


def cut_of(units: int, fp4: bool, down: bool) -> tuple[int, int]:
    """(waves that share a row, loads of each)."""
    best = (0, 0)
    for splits in (8, 4, 2, 1):
        first = 1 if down and splits == units else 2 if fp4 else 8
        for loads in (first, 2, 3, 4) if fp4 else (8, 8, 12, 16):
            if loads * splits < units or (down and loads > 2 and units <= 16):
                continue
            if not best[0] or loads * splits < best[0] * best[1]:
                best = (splits, loads)
    return best


def rows_kernel(product: int, length: int, tiles: int, items: int, wide: bool) -> dict:
    fp4, down = product != UP_BF16, product == DOWN_FP4
    units = (length + 127) // 128 if fp4 else length // 32
    splits, loads = cut_of(units, fp4, down)
    steps = loads * (4 if fp4 else 1)
    full = units == splits * loads and length % 128 == 0
    subs = 8 // splits
    share = subs
    while items * tiles // (2 * share) >= (1024 if fp4 or wide else 2048) and share < 8 * subs:
        share *= 2
    held = 4 if down and steps <= 4 else 8 if steps <= 8 else 12 if steps <= 12 else 16
    full = full and not (down and held == 12)
    if wide:
        columns = {8: 4, 12: 2, 16: 1}[held] if product == UP_BF16 else 2 if down or held <= 8 else 1
    else:
        columns = 2 if down else 1
    batch = 1
    if fp4 and held <= 8:
        batch = (2 if held == 8 else 4) if down else 2 if wide else 4
    if share // subs < batch:
        batch = 1
    return {
        "name": f"experts_rows_kernelILNS0_7ProductE{product}ELi{held}ELb{int(full)}ELi{columns}ELi{batch}EE",
        "columns": columns, "pairs": 8 if down else 16, "splits": splits,
    }


def down_kernel(width: int, many: bool) -> str:
    steps = (width + 31) // 32
    each = (steps + 7) // 8
    held = 2 if each <= 2 else each if each <= 4 else 8
    mode = HALF_STEP if width % 32 else RAGGED if steps % (8 * held) else EXACT
    return f"experts_down{'_many' if many else ''}_kernelILi{held}ELNS0_5StepsE{mode}EE"


def launches(hidden: int, width: int, experts: int, top_k: int, tokens: int, fp4: bool,
             counts: list[int]) -> set[tuple]:
    """(kernel, column tiles of a pass, whether a run takes several passes) of one call.

    `counts` are the pairs of each expert that has any.
    """
    pairs = tokens * top_k
    splits, loads = cut_of(hidden // (128 if fp4 else 32), fp4, False)
    if fp4:
        wide = splits == 8 and loads <= 2 and pairs >= 28 * experts
    else:
        wide = loads <= 12 and pairs >= 8 * experts
    items = pairs if pairs <= experts else experts
    runs = list(counts)
    found = set()
    if pairs > 64:
        most = 16 if not wide else 32 if fp4 else 64
        items = min(experts, pairs) + pairs // most
        runs = [min(most, n - at) for n in counts for at in range(0, n, most)]
        found.add(("experts_sort_kernel", 0, False))

    def rows(kernel: dict) -> None:
        for n in runs:
            left, passes = n, []
            while left > 0:
                for tiles in (4, 2, 1):
                    if tiles == 1 or (kernel["columns"] >= tiles and left > tiles // 2 * kernel["pairs"]):
                        passes.append(tiles)
                        left -= tiles * kernel["pairs"]
                        break
            found.update((kernel["name"], tiles, len(passes) > 1) for tiles in passes)

    rows(rows_kernel(UP_FP4 if fp4 else UP_BF16, hidden, width // 8, items, wide))
    few = tokens * (hidden // 16) <= 1280 and pairs * hidden * (width // 2) <= 10_000_000 * min(top_k, 4)
    if fp4 and pairs <= experts and few:
        found.add(("experts_fp4_tokens_kernel", 0, False))
        return found
    if fp4:
        rows(rows_kernel(DOWN_FP4, width, hidden // 16, items, False))
    else:
        found.update((down_kernel(width, wide), 1, n > 16) for n in runs)
    found.add(("experts_join_kernel", 0, False))
    return found


# hidden, width, experts, pairs (one a token), 4 bits, pairs of each expert that has any;
# the other pairs name no expert, and the other experts have no weights but zeros. Ten
# experts for these 59 pairs make narrow calls, three wide ones over BF16 rows.
MIXED = [36, 20, 3]
CASES = [
    # the up product's row lengths
    *((hidden, width, experts, 59, fp4, MIXED)
      for fp4, width in ((False, 16), (True, 32)) for experts in (10, 3)
      for hidden in (128, 256, 384, 640, 1152, 1536, 2176, 2304, 3200, 3968, 4096)),
    # the BF16 down product's widths: whole rounds of the waves, ragged ones, half a step
    *((128, width, experts, 59, False, MIXED) for experts in (10, 3)
      for width in (144, 320, 400, 496, 512, 528, 608, 720, 768, 784, 800, 976, 1008, 1024, 1056,
                    2048, 2064, 2080, 4080, 4096)),
    # two and four output tiles a workgroup
    *((hidden, width, 64, 64, False, MIXED) for width in (272, 512, 528, 608, 768, 784, 800, 1024, 1056, 2064)
      for hidden in (512, 1024)),
    # the 4-bit down product's
    *((128, width, 10, 59, True, MIXED)
      for width in (32, 96, 160, 256, 384, 480, 512, 640, 960, 992, 1024, 1056, 1152, 1984, 2016, 2048, 2080,
                    2976, 3104, 4064, 4096)),
    # wide calls over 4-bit rows, unsorted and sorted
    *((hidden, 32, 2, 59, True, [39, 20]) for hidden in (1664, 1792, 1920, 2048)),
    *((hidden, 32, 3, 100, True, MIXED) for hidden in (1920, 2048)),
    # several row tiles of 4-bit rows between two barriers
    (256, 256, 1024, 1024, True, MIXED), (384, 32, 64, 800, True, MIXED), (2048, 256, 64, 1800, True, MIXED),
    (1792, 256, 64, 1800, True, MIXED), (2048, 256, 200, 300, True, MIXED), (1920, 256, 200, 300, True, MIXED),
    (128, 2048, 256, 300, True, MIXED), (256, 1920, 256, 300, True, MIXED), (256, 768, 400, 600, True, MIXED),
    (1024, 96, 512, 600, True, MIXED), (1024, 128, 512, 600, True, MIXED), (256, 480, 512, 600, True, MIXED),
    (256, 1024, 512, 600, True, MIXED),
    # 4-bit rows of few tokens, about the most of them in workgroups and in bytes
    (512, 160, 8, 3, True, [2, 1]), (512, 160, 64, 40, True, [20, 3, 1]), (512, 160, 64, 41, True, [20, 3, 1]),
    (128, 4096, 64, 38, True, [20, 3, 1]), (128, 4096, 64, 39, True, [20, 3, 1]),
    (128, 32, 160, 160, True, [90, 3, 1]),
    # sorted runs of 64 and 32 pairs
    (256, 96, 8, 500, False, [100, 70, 17, 16, 1]),
    (256, 96, 8, 500, True, [100, 70, 17, 16, 1]),
]
