"""What the head's loss asks for as workspace (host code, no GPU)."""
import ctypes as C

import pytest

from monarch_muon_amd import _abi

MiB = 1 << 20


def need(T, D, V, piece, train=1, **kw):
    args = dict(tokens=T, vocab=V, width=D, dtype=_abi.BF16, reduction=_abi.CE_MEAN, x_stride=D, w_stride=D,
                piece_tokens=piece, x=4096, w=8192, target=12288, loss=16384, dx=20480, dw=24576)
    return _abi.lib().mmuon_ce_workspace(C.byref(_abi.CeArgs(**{**args, **kw})), train)


@pytest.mark.parametrize("T, D, V, piece", [(4096, 4096, 50304, 2048), (4096, 4096, 50304, 256), (900, 264, 33000, 400)])
def test_sums_of_dw_are_there_only_for_dw(T, D, V, piece):
    """Several pieces keep fp32 sums of dw; a frozen head has none, nor partial sums of them."""
    frozen, whole = need(T, D, V, piece, dw=None), need(T, D, V, piece)
    assert whole - frozen >= 4 * D * V
    codes = piece * (V + 255) // 256 * 256 * 2
    # codes, gathered rows, statistics, the lists; partial sums of the logits or of dx, 256 MiB at most
    rest = piece * (2 * D + V // 8 + 64) + T * 32 + 256 * MiB
    assert frozen <= codes + rest, (frozen / MiB, codes / MiB, rest / MiB)


def test_partial_sums_of_dx_are_there_only_for_dx():
    """200 tokens of 70000 x 520: dx has a few tiles, all split over the vocabulary; the logits and dw none."""
    tiles = 3 * 2 * 42   # 256 x 128 of 520 x 200, 42 parts
    assert need(200, 520, 70000, 200) - need(200, 520, 70000, 200, dx=None) == tiles * 256 * 128 * 4
    assert need(200, 520, 70000, 200, dx=None) == need(200, 520, 70000, 200, dx=None, dw=None)


def test_one_piece_keeps_no_sums():
    """dw of one piece is written as it is made (128 tokens of 45000 x 2048: no tile of it is split)."""
    assert need(128, 2048, 45000, 128) == need(128, 2048, 45000, 128, dw=None)
    assert need(128, 2048, 45000, 128, train=0) == need(128, 2048, 45000, 128, train=0, dx=None, dw=None)
