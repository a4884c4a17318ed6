"""The operators between a layer's projections without a GPU, at the ends of what their entry points allow."""
import ctypes as C
import math

import pytest
import torch

from monarch_muon_amd import _abi, rotary_table

ATTENTION = dict(batch=1, queries=4, keys=4, heads=2, kv_heads=1, dim=64, dtype=_abi.BF16, scale=1.0, q=4096, k=8192, v=12288,
                 lam=16384, o=20480, o1=24576, o2=28672, lse=32768, dout=36864, dq=40960, dk=45056, dv=49152, dlam=53248,
                 workspace=65536, workspace_bytes=1 << 40)


def refusal(fn, args, *more):
    lib = _abi.lib()
    rc = getattr(lib, fn)(C.byref(args), *more, None)
    return rc, lib.mmuon_last_error().decode()


@pytest.mark.parametrize("none", [dict(queries=0), dict(heads=0)])
@pytest.mark.parametrize("missing", [dict(k=0), dict(v=0), dict(k=0, v=0), dict(k=8194)])
def test_keys_gradients_of_no_query_need_keys(none, missing):
    """Their zeros come from a kernel that reads the keys first."""
    rc, why = refusal("mmuon_attention_bwd", _abi.AttentionArgs(**{**ATTENTION, **none, **missing}))
    assert rc == -1 and "q, k or v" in why, why


@pytest.mark.parametrize("rows, code, match", [((1 << 28) - 8, -3, "too many"), ((1 << 28) - 15, -3, "too many"),
                                               ((1 << 28) - 16, -1, "unaligned gradients")])
def test_rows_of_the_backwards_largest_launch(rows, code, match):
    """16 threads to a row, 256 to a workgroup: fewer than 2^32 in all.  (The last case goes on to dk's address.)"""
    sizes = dict(heads=1, keys=1, queries=rows, dk=45058)
    rc, why = refusal("mmuon_attention_bwd", _abi.AttentionArgs(**{**ATTENTION, **sizes}))
    assert rc == code and match in why, why


ROTARY = dict(batch=1, tokens=4, q_heads=32, k_heads=32, dim=128, part=128, dtype=_abi.BF16, table_rows=9, q=4096, k=8192,
              table=12289, q_out=16384, k_out=20480)


@pytest.mark.parametrize("change, code, match", [
    (dict(tokens=1 << 18), -1, "unaligned table"), (dict(tokens=1 << 26), -1, "unaligned table"),
    (dict(tokens=1 << 27), -3, "too many"), (dict(batch=1 << 27, tokens=1), -3, "too many"),
    (dict(q_heads=1 << 24, dim=256, part=2), -3, "too many"), (dict(q_heads=1 << 22, part=2), -1, "unaligned table")])
def test_rotary_takes_long_sequences(change, code, match):
    """2^40 elements of all, and one token's 2^31.  (What is taken goes on to the table's address, which is none.)"""
    rc, why = refusal("mmuon_rotary", _abi.RotaryArgs(**{**ROTARY, **change}), 0)
    assert rc == code and match in why, why


@pytest.mark.parametrize("B, T, H, K, d", [(4, 222563, 96, 24, 72), (2, 259541, 148, 37, 96), (253, 128675, 16, 2, 16), (9, 269351, 100, 25, 8)])
def test_workspace_of_many_keys(B, T, H, K, d):
    """Queries and keys in parts are for calls of few tiles: rounds of workgroups that end a little earlier are not worth
    tens of gigabytes.  What is left are the rows' statistics and their parts of dlam."""
    a = _abi.AttentionArgs(**{**ATTENTION, "batch": B, "queries": T, "keys": T, "heads": H, "kv_heads": K, "dim": d})
    assert _abi.lib().mmuon_attention_workspace(C.byref(a), 1) <= 20 * B * H * T + 4096


@pytest.mark.parametrize("kw", [
    dict(scaling="llama", fast=1.0), dict(scaling="llama", fast=4.0, slow=4.0), dict(scaling="llama", fast=1.0, slow=4.0),
    dict(scaling="llama", slow=math.nan), dict(scaling="yarn", fast=1.0, slow=32.0), dict(scaling="yarn", slow=0.0),
    dict(scaling="yarn", fast=math.nan), dict(scaling="yarn", base=1.0), dict(scaling="yarn", base=0.5)])
def test_a_ramp_over_no_turns_is_refused(kw):
    """A ramp needs turns that it rises over (0 / 0 where a pair stands at both its ends), and one by pairs falling angles."""
    with pytest.raises(ValueError, match="fast|base"):
        rotary_table(64, 128, **{"factor": 2.0, "trained": 512, **kw})
    if "base" not in kw:                       # who has no ramp takes no notice
        assert not rotary_table(64, 128, **{"trained": 512, **kw, "scaling": None}).isnan().any()


@pytest.mark.parametrize("kw", [dict(scaling="llama", slow=0.0), dict(scaling="yarn", fast=1.0, slow=1.0)])
def test_the_narrowest_ramps(kw):
    """From no turn at all, and a step between one pair and the next."""
    table = rotary_table(64, 128, factor=2.0, trained=512, **kw)
    assert table.isfinite().all() and not torch.equal(table, rotary_table(64, 128))
