"""Token pools without a GPU: the page model keeps every page once, and every
entry point refuses bad arguments on the host before anything is launched."""
import ctypes

import numpy as np
import pytest

from oracle.tokens import TokenPoolModel
from parakeet_b200 import _lib

FAKE = 1 << 20   # never dereferenced: the calls under test return before a launch


def make_desc(**kw):
    d = _lib.TokenKVDesc(num_pages=16, num_slots=4, num_layers=2, num_heads=8, num_kv_heads=4,
                         head_dim=64, page_size=16, table_width=4, dtype=_lib.PK_DTYPE_F32)
    for k in ("kv", "page_table", "free_pages", "free_count", "lengths", "held", "scratch", "error"):
        setattr(d, k, FAKE)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.fixture
def pool():
    h = ctypes.c_void_p()
    assert _lib.lib().pk_token_kv_create(ctypes.byref(make_desc()), ctypes.byref(h)) == _lib.PK_OK
    yield h
    _lib.lib().pk_token_kv_destroy(h)


@pytest.mark.parametrize("bad", [dict(kv=None), dict(scratch=None), dict(error=None), dict(dtype=2),
                                 dict(num_pages=0), dict(table_width=0), dict(num_kv_heads=3),
                                 dict(num_kv_heads=0), dict(head_dim=96), dict(head_dim=256),
                                 dict(page_size=12), dict(page_size=4), dict(page_size=512),
                                 dict(num_pages=1 << 28), dict(table_width=1 << 28),
                                 dict(kv=FAKE + 8), dict(num_layers=1 << 28)])
def test_create_refuses(bad):
    h = ctypes.c_void_p()
    assert _lib.lib().pk_token_kv_create(ctypes.byref(make_desc(**bad)),
                                         ctypes.byref(h)) == _lib.PK_EINVAL
    assert not h.value


def test_step_block_layout(pool):
    """The arrays lie behind each other without overlap, masks 8-byte aligned."""
    at = (ctypes.c_int64 * _lib.PK_TOK_OFFSETS)()
    for batch, rows, trees in [(1, 1, 1), (3, 7, 1), (4, 1001, 0), (4, 0, 1)]:
        words = _lib.lib().pk_token_step_words(pool, batch, rows, trees, at)
        n = {_lib.PK_TOK_ROW_START: batch + 1, _lib.PK_TOK_CONTEXT: batch, _lib.PK_TOK_REQUEST: rows,
             _lib.PK_TOK_POSITION: rows, _lib.PK_TOK_SLOT_MAP: rows,
             _lib.PK_TOK_MASK: 2 * rows if trees else 0}
        spans = sorted((at[i], at[i] + k) for i, k in n.items() if k)
        assert spans[0][0] >= 16 and spans[-1][1] <= words
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
        assert at[_lib.PK_TOK_MASK] % 2 == 0
    assert _lib.lib().pk_token_step_words(pool, -1, 1, 0, None) == -1
    assert _lib.lib().pk_token_step_words(pool, 1, -1, 0, None) == -1


def test_calls_refuse(pool):
    lib, E = _lib.lib(), _lib.PK_EINVAL
    begin, end = lib.pk_token_begin_step, lib.pk_token_end_step
    assert begin(None, FAKE, FAKE, 1, None, 1, FAKE, None) == E
    assert begin(pool, None, FAKE, 1, None, 1, FAKE, None) == E
    assert begin(pool, FAKE, None, 1, None, 1, FAKE, None) == E
    assert begin(pool, FAKE, FAKE, 1, None, 1, None, None) == E
    assert begin(pool, FAKE, FAKE, 1, None, 1, FAKE + 4, None) == E      # misaligned block
    assert begin(pool, FAKE, FAKE, 5, None, 1, FAKE, None) == E          # above num_slots
    assert begin(pool, FAKE, FAKE, -1, None, 1, FAKE, None) == E
    assert begin(pool, FAKE, FAKE, 1, None, -1, FAKE, None) == E
    assert begin(pool, FAKE, FAKE, 1, None, (1 << 31) // 8, FAKE, None) == E
    assert begin(pool, FAKE, FAKE, 0, None, 0, None, None) == _lib.PK_OK
    app = lib.pk_token_append
    assert app(pool, 2, 1, FAKE, FAKE, 0, 256, 64, 1, 1, 0, FAKE, None) == E   # past the layers
    assert app(pool, -1, 1, FAKE, FAKE, 0, 256, 64, 1, 1, 0, FAKE, None) == E
    assert app(pool, 0, 1, None, FAKE, 0, 256, 64, 1, 1, 0, FAKE, None) == E
    assert app(pool, 0, 1, FAKE, FAKE + 4, 0, 256, 64, 1, 1, 0, FAKE, None) == E
    assert app(pool, 0, 1, FAKE, FAKE, 0, 255, 64, 1, 1, 0, FAKE, None) == E
    assert app(pool, 0, 1, FAKE, FAKE, 0, 256, 64, 1, 0, 0, FAKE, None) == _lib.PK_OK
    att = lib.pk_token_attention
    assert att(pool, 2, FAKE, 512, 64, 0.1, 1, 1, 0, FAKE, FAKE, 512, 64, None, None) == E
    assert att(pool, 0, None, 512, 64, 0.1, 1, 1, 0, FAKE, FAKE, 512, 64, None, None) == E
    assert att(pool, 0, FAKE, 512, 64, 0.0, 1, 1, 0, FAKE, FAKE, 512, 64, None, None) == E
    assert att(pool, 0, FAKE, 512, 64, -1.0, 1, 1, 0, FAKE, FAKE, 512, 64, None, None) == E
    assert att(pool, 0, FAKE, 512, 64, float("nan"), 1, 1, 0, FAKE, FAKE, 512, 64, None, None) == E
    assert att(pool, 0, FAKE, 511, 64, 0.1, 1, 1, 0, FAKE, FAKE, 512, 64, None, None) == E
    assert att(pool, 0, FAKE, 512, 64, 0.1, 1, 1, 0, FAKE, FAKE, 512, 63, None, None) == E
    assert att(pool, 0, FAKE, 512, 64, 0.1, 1, 1, 0, None, FAKE, 512, 64, None, None) == E
    assert end(pool, None, 1, 1, 0, FAKE, None) == E
    assert end(pool, FAKE, 1, 1, 0, None, None) == E
    assert lib.pk_token_truncate(pool, FAKE, None, 1, None) == E
    assert lib.pk_token_truncate(pool, None, FAKE, 1, None) == E
    assert lib.pk_token_truncate(pool, FAKE, FAKE, 5, None) == E
    assert lib.pk_token_truncate(pool, FAKE, FAKE, 0, None) == _lib.PK_OK


def test_workspace_needed_when_requests_can_be_split():
    """A pool whose requests may be long splits their keys; without a workspace the
    call is refused."""
    lib, h = _lib.lib(), ctypes.c_void_p()
    assert lib.pk_token_kv_create(ctypes.byref(make_desc(table_width=256)), ctypes.byref(h)) == 0
    assert lib.pk_token_attention_workspace(h, 1, 1) > 0
    assert lib.pk_token_attention(h, 0, FAKE, 512, 64, 0.1, 1, 1, 0, FAKE, FAKE, 512, 64, None,
                                  None) == _lib.PK_EINVAL
    lib.pk_token_kv_destroy(h)


def test_model_keeps_every_page_once_and_restores_the_stack():
    rng = np.random.default_rng(0)
    m = TokenPoolModel(6, 200, 40, 8, order=rng.permutation(40))
    for _ in range(300):
        slots = rng.permutation(6)[: rng.integers(1, 7)]
        counts = rng.integers(0, 20, len(slots))
        before = list(m.stack)
        lengths = m.lengths[slots].copy()
        held = m.held.copy()
        step = m.begin_step(slots, counts, int(counts.sum()))
        if rng.random() < 0.5 and all(held == -(-m.lengths // 8)):
            m.truncate(slots, lengths)          # cut back: no trace
            assert m.stack == before
        else:
            ok = step["context"] >= 0
            m.end_step(step, np.where(ok, counts - 1, -1))
            cut = rng.random(len(slots)) < 0.3
            m.truncate(slots, np.where(cut, 0, m.lengths[slots]))
        pages = m.table[m.table >= 0].tolist() + m.stack
        assert sorted(pages) == list(range(40))
