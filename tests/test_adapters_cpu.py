"""The adapters' host-side refusals (no GPU: nothing is launched)."""
import pytest

from parakeet_b200 import _lib

FAKE = 1 << 20


def call(M=8, N=128, K=64, lda=64, ldw=64, ldc=128, epi=0, R=None, ldr=0, bias=None, rank=16, n=4,
         A=FAKE, W=FAKE, C=FAKE, down=FAKE, up=FAKE, plan=FAKE, ws=FAKE, err=FAKE):
    return _lib.lib().pk_adapter_gemm(A, lda, W, ldw, M, N, K, C, ldc, epi, R, ldr, bias, 1.0, down,
                                      up, rank, n, None, plan, ws, err, None)


@pytest.mark.parametrize("bad", [
    dict(M=-1), dict(M=(1 << 20) + 1), dict(N=96), dict(K=96), dict(K=0), dict(rank=0), dict(rank=12),
    dict(rank=136), dict(n=0), dict(n=8193), dict(epi=5), dict(epi=-1), dict(lda=56), dict(lda=65),
    dict(ldw=56), dict(ldc=120), dict(A=None), dict(W=None), dict(C=None), dict(down=None),
    dict(up=None), dict(plan=None), dict(ws=None), dict(err=None), dict(A=FAKE + 8),
    dict(down=FAKE + 2), dict(up=FAKE + 2), dict(plan=FAKE + 4), dict(ws=FAKE + 8), dict(epi=2),
    dict(epi=3, R=FAKE, ldr=64), dict(epi=2, R=FAKE + 2, ldr=128), dict(epi=4)])
def test_gemm_refuses(bad):
    assert call(**bad) == _lib.PK_EINVAL


def test_empty_calls_are_fine():
    lib = _lib.lib()
    assert call(M=0) == _lib.PK_OK
    assert lib.pk_adapter_plan(None, 0, 4, None, None, None) == _lib.PK_OK


def test_plan_refuses():
    lib, E = _lib.lib(), _lib.PK_EINVAL
    assert lib.pk_adapter_plan(FAKE, -1, 4, FAKE, FAKE, None) == E
    assert lib.pk_adapter_plan(FAKE, 4, 0, FAKE, FAKE, None) == E
    assert lib.pk_adapter_plan(FAKE, 4, 8193, FAKE, FAKE, None) == E
    assert lib.pk_adapter_plan(None, 4, 4, FAKE, FAKE, None) == E
    assert lib.pk_adapter_plan(FAKE, 4, 4, FAKE + 4, FAKE, None) == E
    assert lib.pk_adapter_plan(FAKE, 4, 4, FAKE, None, None) == E


def test_sizes():
    """The plan holds the sorted rows padded to 128-row tiles, a flag and, at most, a pair
    (of 8 words) for each adapter in use and one more for each tile."""
    lib = _lib.lib()
    for rows, n in [(1, 1), (128, 5), (129, 8192), (6720, 64)]:
        tiles = -(-rows // 128)
        words = lib.pk_adapter_plan_words(rows, n)
        need = tiles * 128 + tiles + 2 + 8 * (tiles + min(rows, n))
        assert need <= words <= need + 3
        assert lib.pk_adapter_workspace(rows, 64, 16) == tiles * 128 * (64 + 16) * 2
    assert lib.pk_adapter_plan_words(-1, 1) == -1 and lib.pk_adapter_plan_words(1, 0) == -1
    assert lib.pk_adapter_workspace(1, 64, 0) == -1
