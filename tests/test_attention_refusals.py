"""What the entry points of the attention operators refuse before anything is enqueued (no GPU: the pointers are never followed), and the host's side of
the rotation's table."""

import ctypes
import math
import os

import pytest

from tilefish_b200 import TilefishPreconditionError, _native as N
from tilefish_b200 import attention as A

needs_library = pytest.mark.skipif(not os.path.exists(N.LIB_PATH), reason="library not built here")
AT = 1 << 20  # an aligned address that nothing follows


def cache(**kwargs):
    fields = dict(k=AT, v=2 * AT, k_scale=None, v_scale=None, pages=4, page_size=16, kv_heads=2, head_dim=64, stride_page=2048, stride_head=1024, stride_slot=64, dtype=0, reserved=0)
    fields.update(kwargs)
    return N.PagedCacheDescriptor(**fields)


def rotary(**kwargs):
    a = dict(x=AT, dtype=0, tokens=4, heads=2, head_dim=64, xt=128, xh=64, positions=AT, bits=64, turns=AT, rot=64, layout=0, magnitude=1.0, inverse=0, out=2 * AT, ot=128, oh=64, stream=None)
    a.update(kwargs)
    return N.load().tf_rotary(*a.values())


def append(c=None, **kwargs):
    a = dict(k=AT, kt=128, kh=64, v=AT, vt=128, vh=64, tokens=4, tables=AT, table_rows=2, table_cols=3, table_stride=3, positions=AT, bits=32, rows=None, q=AT, q_heads=4, qt=256, qh=64,
             q_out=2 * AT, ot=256, oh=64, turns=AT, rot=64, layout=1, magnitude=1.0, stream=None)
    a.update(kwargs)
    c = c or cache()
    return N.load().tf_cache_append(ctypes.addressof(c), *a.values())


def attend(c=None, **kwargs):
    a = dict(q=AT, qt=256, qh=64, seqs=2, queries=2, q_heads=4, tables=AT, table_cols=3, table_stride=3, lengths=AT, counts=None, scale=0.125, window=0, out=2 * AT, ot=256, oh=64, lse=None,
             workspace=AT, workspace_bytes=1 << 40, stream=None)
    a.update(kwargs)
    c = c or cache()
    return N.load().tf_paged_attention(ctypes.addressof(c), *a.values())


BAD, ODD, NOT = N.TF_ERR_INVALID_ARGUMENT, N.TF_ERR_ALIGNMENT, N.TF_ERR_UNSUPPORTED


@needs_library
@pytest.mark.parametrize("status,change", [(BAD, {"x": None}), (BAD, {"out": None}), (BAD, {"positions": None}), (BAD, {"turns": None}), (BAD, {"dtype": 2}), (BAD, {"tokens": -1}),
                                           (BAD, {"heads": 0}), (BAD, {"head_dim": 2048}), (BAD, {"rot": 63}), (BAD, {"rot": 66}), (BAD, {"rot": 0}), (BAD, {"layout": 2}),
                                           (BAD, {"bits": 16}), (ODD, {"x": AT + 1}), (ODD, {"out": AT + 2, "dtype": 1}), (ODD, {"positions": AT + 4}), (ODD, {"turns": AT + 4})])
def test_rotary_refuses(status, change):
    assert rotary(**change) == status and N.last_error()


BAD_CACHES = [(BAD, {"k": None}), (BAD, {"v": None}), (BAD, {"dtype": 2}), (BAD, {"pages": 0}), (BAD, {"pages": 1 << 31}), (BAD, {"page_size": 0}), (BAD, {"kv_heads": 0}),
              (NOT, {"head_dim": 40}), (NOT, {"head_dim": 272}), (NOT, {"head_dim": 0}), (ODD, {"k": AT + 8}), (ODD, {"v": AT + 8}), (ODD, {"stride_slot": 68}), (ODD, {"stride_page": -2048}),
              (ODD, {"stride_head": 1032, "dtype": 1}), (BAD, {"k_scale": AT}), (ODD, {"v_scale": AT + 2, "dtype": 1})]


@needs_library
@pytest.mark.parametrize("status,change", BAD_CACHES)
def test_a_bad_cache_is_refused(status, change):
    assert append(cache(**change)) == status and N.last_error()
    assert attend(cache(**change)) == status and N.last_error()


@needs_library
@pytest.mark.parametrize("status,change", [(BAD, {"k": None}), (BAD, {"v": None}), (BAD, {"tables": None}), (BAD, {"positions": None}), (BAD, {"q": None}), (BAD, {"q_out": None}),
                                           (BAD, {"q": None, "q_out": None}), (BAD, {"tokens": -1}), (BAD, {"tokens": 3}), (BAD, {"table_rows": 0}), (BAD, {"table_cols": 0}),
                                           (BAD, {"q_heads": -1}), (BAD, {"bits": 8}), (BAD, {"layout": -1}), (BAD, {"rot": 66}), (BAD, {"turns": None}), (BAD, {"rot": 0}),
                                           (ODD, {"k": AT + 2}), (ODD, {"v": AT + 4}), (ODD, {"q": AT + 8}), (ODD, {"q_out": AT + 8}), (ODD, {"kt": 100}), (ODD, {"oh": 4}), (ODD, {"tables": AT + 2}),
                                           (ODD, {"rows": AT + 1}), (ODD, {"positions": AT + 2})])
def test_append_refuses(status, change):
    assert append(**change) == status and N.last_error()


@needs_library
@pytest.mark.parametrize("status,change", [(BAD, {"q": None}), (BAD, {"out": None}), (BAD, {"tables": None}), (BAD, {"lengths": None}), (BAD, {"seqs": -1}), (BAD, {"queries": 0}),
                                           (BAD, {"q_heads": 0}), (BAD, {"q_heads": 3}), (BAD, {"table_cols": 0}), (BAD, {"window": -1}), (BAD, {"seqs": 1 << 31}),
                                           (ODD, {"q": AT + 8}), (ODD, {"out": AT + 8}), (ODD, {"workspace": AT + 8}), (ODD, {"qt": 100}), (ODD, {"oh": 12}), (ODD, {"tables": AT + 2}), (ODD, {"lengths": AT + 1}),
                                           (ODD, {"counts": AT + 2}), (ODD, {"lse": AT + 2}), (BAD, {"scale": math.inf}), (BAD, {"scale": math.nan})])
def test_attention_refuses(status, change):
    assert attend(**change) == status and N.last_error()


@needs_library
def test_attention_refuses_a_small_workspace():
    need = N.load().tf_paged_attention_workspace_bytes(2, 2, 4, 2, 64, 0, 48)
    assert need > 0
    assert attend(workspace_bytes=need - 1) == N.TF_ERR_WORKSPACE and attend(workspace=None) == N.TF_ERR_WORKSPACE and str(need) in N.last_error()


@needs_library
def test_nothing_to_do_is_no_error():
    assert rotary(tokens=0) == append(tokens=0) == attend(seqs=0) == N.TF_OK
    assert N.load().tf_paged_attention_workspace_bytes(0, 0, 4, 2, 64, 0, 16) == -1


def test_turns_are_the_exact_fraction_of_a_turn():
    two_pi = 2 * math.pi
    for f in (1.0, 0.1, 1e-6, 3.0, 100.0, -0.25):
        (turns,) = A._turns([f])
        assert -(2**63) <= turns < 2**63
        # math.fmod of a 64-bit product is as near as 64-bit floats get
        assert abs(((turns / 2**64) - f / two_pi + 0.5) % 1.0 - 0.5) < 1e-15 * max(1.0, abs(f))
    (turns,) = A._turns([math.pi / 2])  # the double nearest to pi / 2 is 6.1e-17 rad below it
    assert abs(turns - 2**62) < 2**64 * 1e-17


def test_frequencies():
    inv, magnitude = A.rotary_frequencies(64)
    assert len(inv) == 32 and inv[0] == 1.0 and magnitude == 1.0 and abs(inv[16] - 0.01) < 1e-15
    linear, _ = A.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert linear == [f / 4 for f in inv]
    ntk, _ = A.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == inv[0] and abs(ntk[-1] * 4 / inv[-1] - 1) < 1e-12
    for scaling in ("bands", "yarn"):
        f, magnitude = A.rotary_frequencies(64, scaling=scaling, factor=4.0, length=4096)
        assert f[0] == inv[0] and abs(f[-1] * 4 / inv[-1] - 1) < 1e-12 and all(a / 4 - 1e-18 <= b <= a for a, b in zip(inv, f)) and f == sorted(f, reverse=True)
    assert abs(magnitude - (0.1 * math.log(4.0) + 1)) < 1e-15


@pytest.mark.parametrize("kwargs", [{"rot": 0}, {"rot": 7}, {"rot": 64, "scaling": "cubic"}, {"rot": 64, "scaling": "linear", "factor": 0.5}, {"rot": 64, "scaling": "yarn", "factor": 2.0},
                                    {"rot": 64, "scaling": "bands", "factor": 2.0, "length": 10, "low": 4.0}, {"rot": 64, "base": 0.0}])
def test_frequencies_refuse(kwargs):
    with pytest.raises(TilefishPreconditionError):
        A.rotary_frequencies(**kwargs)


def test_a_table_refuses():
    for args, kwargs in (([[1.0]], {"layout": "pairs"}), ([[]], {}), ([[math.nan]], {}), ([[2.0**33]], {}), ([[1.0]], {"magnitude": math.inf}), ([[1.0]], {"magnitude": 1e39}), ([[1.0] * 513], {})):
        with pytest.raises(TilefishPreconditionError):
            A.RotaryTable(*args, device="cpu", **kwargs)
    assert A.RotaryTable([1.0, 0.5], device="cpu").rot == 4


def test_cpu_tensors_are_refused():
    import torch

    table = A.RotaryTable([1.0], device="cpu")
    with pytest.raises(TilefishPreconditionError) as e:
        A.rotary(torch.zeros(1, 1, 2, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64), table)
    assert e.value.kind == "device"
    with pytest.raises(TilefishPreconditionError) as e:
        A.PagedCache(*(torch.zeros(1, 1, 16, 64, dtype=torch.bfloat16) for _ in range(2)))
    assert e.value.kind == "device"
