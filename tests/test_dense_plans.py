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
