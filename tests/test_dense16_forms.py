"""That the cases of test_gpu_dense16_forms.py, and a few more here, run every form of mf_project and mf_bf16_experts.  The rules of projection.hip and
bf16_experts.hip stand here once more as plain arithmetic for a card of 256 units, the tiles' costs read from projection.hip itself: where a
change of them moves a case to another form, it fails here, on the CPU."""
import os
import re

import numpy as np
import pytest

from test_gpu_dense16_forms import EXPERTS, PROJECT, test_projection_shapes as run_projection


def source(name):
    return open(os.path.join(os.path.dirname(__file__), "..", "mference_amd", "csrc", name)).read()


SOURCE = source("projection.hip")
SHAPES = [(int(a), int(b), np.float32(c), np.float32(d), np.float32(e), int(f), g == "true")
          for a, b, c, d, e, f, g in re.findall(r"\{(\d+), (\d+), ([\d.]+)f, ([\d.]+)f, ([\d.]+)f, (\d+), (true|false)\}", SOURCE)]
# shape's number: tokens, rows of W, stages of its tiles
LAUNCHED = {int(k): (int(a), int(b), int(c)) for k, a, b, c in re.findall(r"case (\d+): return launch_tiles<(\d+), (\d+), \d+, \d+, \d+, (\d+), GATED", SOURCE)}
CUS = 256


def up(a, b):
    return -(-a // b)


def most_parts():
    count, = re.findall(r"kMostParts = (\d+);", SOURCE)
    size, shift = re.findall(r"kMostPartBytes = (\d+)u << (\d+);", SOURCE)[0]
    return int(count), int(size) << int(shift)


def project_form(t, n, m, gated):
    """("rows", rows of W a workgroup, waves, pieces of eight rows of x) or ("tiles", (tokens, rows of W, stages), parts of the sum)"""
    rows, aligned = 2 * m if gated else m, n % 8 == 0  # (of tensors that lie as the tests' do)
    if t <= 16:
        blocks = up(m, 16)
        rounds = up(blocks, CUS)
        few = 16 if rounds == 1 else up(m, CUS * rounds)
        return "rows", few, 4 if gated or blocks < CUS else 2, 1 if t <= 8 else 2
    parts_most, bytes_most = most_parts()
    blocks = up(n, 64)
    workspace = not (n < 512 or rows >= 32 * CUS)
    best, parts, least = 0, 1, np.float32(3.4e38)
    for k, (tokens, wide, block, block_many, fixed, a_cu, unaligned) in enumerate(SHAPES):
        if not aligned and not unaligned:
            continue
        tiles, p = up(t, tokens) * up(rows, wide), 1
        while p <= (parts_most if workspace else 1):
            size, rounds = 4 * p * t * rows, up(tiles * p, CUS * a_cu)
            if p > 1 and (tiles * p > CUS or blocks // p < 4 or size > bytes_most):
                break
            us = fixed + np.float32(rounds * up(blocks, p)) * (block_many if tiles * p > 2 * CUS else block)
            if p > 1:
                us += np.float32(3.5) + np.float32(size) / np.float32(2e6)
            if us < least:
                least, best, parts = us, k, p
            p *= 2
    return "tiles", LAUNCHED[best], up(blocks, up(blocks, parts))


def experts_form(t, d, f, experts, top_k, shared_f):
    """(routes a tile, rows of a workgroup, groups or parts of the second launch)"""
    if t <= 8:
        rounds = up(d, CUS * 16)
        rows = min(max(up(d, CUS * rounds), 4), 16)
        instance, routes = 8 if rows <= 8 else 16, t * top_k
        live, longest, parts = min(experts, routes), up(max(f, shared_f), 64), 1
        while parts < 4 and live * parts < 16 and parts * 2 * (routes + (t if shared_f else 0)) * instance <= 4096 and longest > parts:
            parts *= 2
        return 8, rows, parts
    groups = 1
    while groups < 4 and d * groups < CUS * 20:
        groups *= 2
    rounds = up(d * groups, CUS * 32)
    return 16, up(min(max(up(d * groups, CUS * rounds), 4), 32), 4) * 4, groups



# what the rules above are in the sources: a change there is one to make here too
RULES = {
    "projection.hip": (
        "if (t <= 16 || n < 512 || rows >= 32ull * device_cu_count()) return 0;",
        "const uint32_t blocks = (a.m + 15) / 16, rounds = (blocks + cus - 1) / cus, few = rounds == 1 ? 16 : (a.m + cus * rounds - 1) / (cus * rounds);",
        "if (GATED || blocks < cus) return a.t <= 8 ? launch_rows<GATED, ALIGNED, 4, 3, 1>(s, a, few) : launch_rows<GATED, ALIGNED, 4, 3, 2>(s, a, few);",
        "rounds = (tiles * p + cus * h.a_cu - 1) / (cus * h.a_cu);",
        "if (p > 1 && (tiles * p > cus || blocks / p < 4 || bytes > kMostPartBytes)) break;",
        "float us = h.fixed + static_cast<float>(rounds * ((blocks + p - 1) / p)) * (tiles * p > 2 * cus ? h.block_many : h.block);",
        "if (p > 1) us += 3.5f + static_cast<float>(bytes) / 2e6f;"),
    "bf16_experts.hip": (
        "while (groups < 4 && p.d * groups < device_cu_count() * 20) groups *= 2;",
        "const uint32_t rounds = (d * groups + cus * most - 1) / (cus * most);",
        "return std::min(std::max((d * groups + cus * rounds - 1) / (cus * rounds), 4u), most);",
        "while (cut.parts < 4 && a.most_live() * cut.parts < 2 * WAVES && cut.parts * 2 * rows * ROWS <= 4096 && longest > cut.parts) cut.parts *= 2;",
        "const uint32_t rows = rows_of_workgroup(p.d, 1, 16, cus);",
        "return rows <= 8 ? launch_down<8, 1, 4, 8>(s, a, rows, 1) : launch_down<16, 1, 4, 8>(s, a, rows, 1);",
        "return launch_down<32, 2, 4, 4>(s, a, (rows_of_workgroup(p.d, groups, 32, cus) + 3) / 4 * 4, groups);"),
}


@pytest.mark.parametrize("name", RULES)
def test_the_rules_are_the_sources(name):
    text = source(name)
    for line in RULES[name]:
        assert line in text, line


def test_the_shapes_are_the_launched():
    assert len(SHAPES) == 10 and sorted(LAUNCHED) == list(range(10))
    for k, shape in enumerate(SHAPES):
        assert LAUNCHED[k][:2] == shape[:2]


ROWS_2, ROWS_4 = ("rows", 9, 2, 1), ("rows", 9, 4, 1)
PROJECT_FORMS = [
    ROWS_2, ROWS_4, ROWS_2, ROWS_4,
    ("rows", 9, 2, 2), ("rows", 9, 4, 2), ("rows", 9, 2, 2), ("rows", 12, 2, 2), ("rows", 11, 4, 1), ROWS_2,
    *[("tiles", (32, 32, 4), p) for p in (13, 15, 14, 8, 4, 2, 2)],
    *[("tiles", (32, 64, 4), p) for p in (1, 1, 4, 8)],
    *[("tiles", (64, 64, 4), p) for p in (1, 1, 2, 8, 4, 15)],
    *[("tiles", (64, 128, 3), p) for p in (1, 1, 4, 4)],
    *[("tiles", (128, 128, 2), 1)] * 4,
    *[("tiles", (128, 128, 3), p) for p in (1, 1, 4, 4)],
    *[("tiles", (128, 192, 3), p) for p in (1, 1, 2, 4)],
    *[("tiles", (256, 128, 3), 1)] * 2, *[("tiles", (256, 192, 2), 1)] * 2, *[("tiles", (256, 256, 2), 1)] * 2,
]
MORE = [  # t, n, m, gated: forms that the cases there leave out
    (3, 2048, 512, 0), (2, 1001, 129, 0), (16, 256, 128, 0), (10, 1001, 129, 0),  # few rows of a small W: four waves
    (9, 512, 4100, 1),  # gated, 9 to 16 rows, whole 16 bytes
    (20, 1001, 96, 0), (20, 8199, 33, 0),  # 32 x 32 of rows at any address
    (5000, 1001, 2048, 1),
]
MORE_FORMS = [
    ("rows", 16, 4, 1), ("rows", 16, 4, 1), ("rows", 16, 4, 2), ("rows", 16, 4, 2), ("rows", 9, 4, 2), ("tiles", (32, 32, 4), 1), ("tiles", (32, 32, 4), 15),
    ("tiles", (128, 128, 2), 1),
]
EXPERTS_FORMS = [(8, 10, 1), (8, 9, 2), (8, 4, 4), (8, 11, 1), (16, 24, 1), (16, 20, 1), (16, 24, 2), (16, 20, 2), (16, 24, 2), (16, 12, 4), (16, 16, 4), (16, 4, 4), (16, 4, 4)]


def test_every_projection_runs_in_the_form_that_it_is_there_for():
    assert [project_form(*c) for c in PROJECT] == PROJECT_FORMS
    assert [project_form(*c) for c in MORE] == MORE_FORMS


def test_every_form_of_a_projection_has_a_case():
    seen = {(form[:1] + form[2:] if form[0] == "rows" else form[:2] + (form[2] > 1,)) + (bool(gated), n % 8 == 0)
            for (t, n, m, gated), form in zip(PROJECT + MORE, PROJECT_FORMS + MORE_FORMS)}
    rows = {("rows", waves, pieces, gated, aligned) for waves in (2, 4) for pieces in (1, 2) for gated in (False, True) for aligned in (False, True) if waves == 4 or not gated}
    assert rows <= seen
    tiles = {("tiles", LAUNCHED[k], gated, aligned) for k, shape in enumerate(SHAPES) for gated in (False, True) for aligned in ((False, True) if shape[6] else (True,))}
    assert {v[:2] + v[3:] for v in seen if v[0] == "tiles"} == tiles
    assert {(v[2], v[3]) for v in seen if v[0] == "tiles"} == {(p, g) for p in (False, True) for g in (False, True)}  # one part and several, gated and not


def test_every_layer_of_experts_runs_in_the_form_that_it_is_there_for():
    assert [experts_form(*c) for c in EXPERTS] == EXPERTS_FORMS
    assert {(rows <= 8) for tile, rows, _ in EXPERTS_FORMS if tile == 8} == {False, True}
    assert {parts for tile, _, parts in EXPERTS_FORMS if tile == 8} == {1, 2, 4} == {groups for tile, _, groups in EXPERTS_FORMS if tile == 16}


@pytest.mark.gpu
@pytest.mark.parametrize("t, n, m, gated", MORE)
def test_more_projection_shapes(gpu, t, n, m, gated):
    run_projection(gpu, t, n, m, gated)
