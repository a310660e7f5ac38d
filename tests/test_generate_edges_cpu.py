"""What the entry points for generating text say about their memory, without a GPU."""
import pytest

from ceo_amd import _lib

DTYPES = {14: 2, 2: 2, 0: 4}


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


@pytest.mark.parametrize("dt", DTYPES)
def test_products_of_many_rows_have_room_for_their_tokens(L, dt):
    """Only up to 32 rows are quantised by the product's kernel: more need bytes for each of them and a scale."""
    for k in (1, 64, 128, 129, 1000, 1024, 1025, 4096, 4097, 8200, 131072):
        kp = -(-k // 128) * 128
        for n in (1, 16, 1024, 16384, 16385, 50257):
            for m in (1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 34, 63, 64, 65, 256, 1000, 16384):
                size = L.linear_int8_workspace_size(m, k, n, dt)
                assert size == 0 and m <= 32 or size >= -(-m // 16) * 16 * kp + 4 * m, (m, k, n)
                if size == 0:
                    assert m <= (32 if dt else 16) if kp <= 1024 else m <= 8 and dt and kp <= 4096


def test_selection_asks_for_what_it_uses(L):
    """A slice is 16384 logits of 2 bytes or 8192 of 4 where there are many rows, with a place for each selected of 8
    bytes and 8 more; a few rows' slices are 8 to a compute unit at most."""
    size = L.beam_select_workspace_size
    assert size(2500, 8, 128003, 64) <= 20000 * (128003 // 8192 + 2) * (8 + 8 * 64)
    assert size(64, 8, 50257, 8) <= 512 * (50257 // 8192 + 2) * 72
    for batch in (1, 3, 100):
        assert size(batch, 4, 1 << 20, 4) <= (4 * batch * 130 + 8 * 512 + 4 * batch) * 40
    assert size(0, 4, 50257, 4) == 0


def test_states_in_place_take_the_library_s_steps(L):
    """The wrapper's limit is the library's; without a token nothing is launched and nothing copied."""
    from ceo_amd import efla

    assert efla.STEP_TOKENS == L.efla_chunk_step_tokens() >= 1
    st = 1 << 20
    assert L.efla_chunk_fwd_hip(16, 16, 16, 16, st, 16, st, None, 2, 0, 2, 2, 64, 64, 64, 14, None, 0, 0, None) == 0


def test_selection_s_workspace_is_enough_for_less(L):
    """Sized for the most texts, beams, tokens and selected, it is enough for fewer of each."""
    size = L.beam_select_workspace_size
    for vocab in (700, 9000, 50257, 128003, 1 << 20):
        for beams, n in ((1, 1), (4, 4), (4, 40), (17, 3), (64, 64)):
            last = 0
            for batch in list(range(1, 700)) + [1000, 1023, 1024, 1025, 2047, 2048, 2049, 5000]:
                got = size(batch, beams, vocab, n)
                assert got >= last, (batch, beams, vocab, n)
                last = got
    for batch in (1, 3, 16, 64, 700):
        last = [0] * 3
        for step in range(1, 65):
            got = [size(batch, 20, 700 * step * step, 5), size(batch, step, 50257, 5), size(batch, 20, 5000, step)]
            assert all(a >= b for a, b in zip(got, last)), (batch, step)
            last = got
