"""How linear layers size their tiles (host arithmetic, no GPU)."""
import random

from fast_b200 import runtime

PAIRS = 74


def _tiles(rows, width, m_tiles):
    return -(-(-(-rows // 32) * 32) // width) * m_tiles


def test_token_tiles_of_one_matrix_need_no_more_rounds_than_full_ones():
    C, r = runtime.ext(), random.Random(1)
    narrower = 0
    for _ in range(4000):
        rows, m_tiles, kb = int(129 * 64 ** r.random()), int(1 + 200 * r.random() ** 3), int(1 + 250 * r.random() ** 2)
        n = C.tok_dense_tile(rows, m_tiles, kb, PAIRS)
        assert n % 32 == 0 and 64 <= n <= 256
        full, mine = (-(-_tiles(rows, w, m_tiles) // PAIRS) for w in (256, n))
        assert mine <= full
        narrower += n < 256
    assert narrower > 400
    for rows, m_tiles in ((1 << 30, 1), (129, 1 << 16), (1 << 20, 1 << 10)):   # many rounds: full tiles, and no overflow
        assert C.tok_dense_tile(rows, m_tiles, 64, PAIRS) == 256


def test_token_tiles_that_were_measured():
    C = runtime.ext()
    for rows, inputs, outputs, want in ((1235, 1000, 2760, 224), (600, 4096, 4096, 160), (1500, 8192, 2048, 192), (500, 7168, 4096, 128), (700, 2048, 7168, 160), (1024, 4096, 4096, 256), (3000, 256, 3000, 256)):
        assert C.tok_dense_tile(rows, -(-outputs // 256), -(-inputs // 64), PAIRS) == want


def _few(T, columns, inputs, swiglu=False, sms=148):
    return runtime.ext().few_plan(T, columns, -(-inputs // 64), swiglu, sms)


def test_plans_for_few_tokens_cover_them_and_fit_an_sm():
    r, seen = random.Random(2), set()
    for _ in range(4000):
        T, columns, blocks, swiglu = int(1024 ** r.random()), 128 * int(500 ** r.random()), int(1 + 300 * r.random() ** 2), r.random() < 0.3
        tiles, token_tiles, n, parts, stages, smem = runtime.ext().few_plan(T, columns, blocks, swiglu, 148)
        per_tile = 64 if swiglu else 128
        assert (tiles - 1) * per_tile < columns <= tiles * per_tile
        assert n % 16 == 0 and 16 <= n <= 128 and (token_tiles - 1) * n < T <= token_tiles * n
        assert parts in (1, 2, 4, 8) and 1 <= parts <= blocks and 1 <= stages <= 12
        ctas, sums = tiles * token_tiles * parts, n * 128 * 4
        assert smem <= (220 if ctas <= 148 else 110) * 1024
        assert smem >= max(stages * (16384 + 128 * n), sums) + 1024 and (parts == 1 or n > 64 or smem >= stages * (16384 + 128 * n) + sums + 1024)
        seen.add((parts, n > 64, ctas <= 148))
    assert {(1, False, True), (1, True, True), (1, True, False), (2, False, True), (2, True, True), (4, False, True), (4, True, True), (8, False, True), (8, False, False)} <= seen


def test_plans_for_few_tokens_that_were_measured():
    for T, inputs, columns, want in ((1, 4096, 4096, 8), (1, 2048, 7168, 2), (1, 4096, 14336, 1), (64, 4096, 4096, 4), (128, 1024, 4096, 2), (256, 4096, 4096, 2), (512, 2048, 4096, 1)):
        assert _few(T, columns, inputs)[3] == want
    assert _few(1, 2048, 7168, swiglu=True)[3] == 8
