"""What the paged serving wrappers hand to the C entries at the edges of what they take, on CPU tensors: the entries are
replaced by ones that keep the packed arguments, and nothing is launched."""

from __future__ import annotations

import pytest
import torch

from torch.autograd import forward_ad

import kernels
from kernels import paged_attention as attention_mod, paged_kv as append_mod
from kernels.paged_attention import paged_attention
from kernels.paged_kv import paged_kv_append
from serve.paged_layer import PagedAttentionLayer
from test_paged_refusals import APPEND, ATTEND, _c_attend

I, BF = torch.int32, torch.bfloat16


@pytest.fixture
def packed(monkeypatch):
    """The fields of the last call of an entry, by name."""
    seen = {}

    class Library:
        def mlsx_paged_attention_ws(self, args):
            return 0

        def mlsx_paged_attention(self, args, *_):
            seen.update(zip(ATTEND, attention_mod._ARGS.unpack(args)))
            return 0

        def mlsx_paged_append(self, args, *_):
            seen.update(zip(APPEND, append_mod._ARGS.unpack(args)))
            return 0

    monkeypatch.setattr(kernels, "lib", lambda: Library())
    for mod in (attention_mod, append_mod):
        monkeypatch.setattr(mod, "one_device", lambda fn, *tensors: 0)
        monkeypatch.setattr(mod, "_raw_stream", lambda index: 0)
    return seen


def _call(kp, vp, heads, write, dtype=BF):
    n, D = 4, kp.shape[3]
    tab, lens = torch.zeros(n, 3, dtype=I), torch.ones(n, dtype=I)
    if write:
        k = torch.zeros(n, kp.shape[1], D, dtype=dtype)
        return paged_kv_append(None, k, k.clone(), kp, vp, tab, lens)
    return paged_attention(torch.zeros(n, heads, D, dtype=dtype), kp, vp, tab, lens)


def _pair(make):
    return make(), make()


READ_ONLY = [  # views whose elements share memory, with their strides
    (lambda: torch.zeros(8, 1, 16, 64, dtype=BF).expand(-1, 4, -1, -1), (1024, 0, 64)),
    (lambda: torch.zeros(8, 4, 1, 64, dtype=BF).expand(-1, -1, 16, -1), (256, 64, 0)),
    (lambda: torch.zeros(1, 4, 16, 64, dtype=BF).expand(8, -1, -1, -1), (0, 1024, 64)),
    (lambda: torch.zeros(99999, dtype=BF).as_strided((8, 4, 16, 64), (1024, 256, 64, 1)), (1024, 256, 64)),
]


@pytest.mark.parametrize("make,strides", READ_ONLY)
def test_views_that_share_memory_are_read_with_their_strides(packed, make, strides):
    _call(*_pair(make), 4, False)
    assert tuple(packed[f] for f in ("kv_sb", "kv_sh", "kv_st")) == strides


@pytest.mark.parametrize("make,strides", READ_ONLY)
def test_views_that_share_memory_are_not_written(packed, make, strides):
    with pytest.raises(ValueError, match="share memory"):
        _call(*_pair(make), 4, True)
    assert not packed


@pytest.mark.parametrize("write", [False, True])
@pytest.mark.parametrize("strides", [(1024, 256, 32, 1), (4096, 32, 128, 1)])
def test_rows_that_overlap_are_refused(packed, write, strides):
    with pytest.raises(ValueError):
        _call(*_pair(lambda: torch.zeros(99999, dtype=BF).as_strided((8, 4, 16, 64), strides)), 4, write)
    assert not packed


@pytest.mark.parametrize("write", [False, True])
@pytest.mark.parametrize("make,strides", [
    (lambda: torch.zeros(8, 16, 4, 64, dtype=BF).transpose(1, 2), (4096, 64, 256)),  # token-major
    (lambda: torch.zeros(4, 8, 16, 64, dtype=BF).transpose(0, 1), (1024, 8192, 64)),  # a head at a time
    (lambda: torch.zeros(8, 2, 4, 16, 64, dtype=BF)[:, 1], (8192, 1024, 64)),  # K and V of a block side by side
    (lambda: torch.zeros(8, 1, 16, 64, dtype=BF).as_strided((8, 1, 16, 64), (1024, 3, 64, 1)), (1024, 64, 64)),  # one head: its
    (lambda: torch.zeros(8, 4, 1, 64, dtype=BF).as_strided((8, 4, 1, 64), (256, 64, 0, 1)), (256, 64, 64)),  # .. stride is none
])
def test_orders_of_a_pool(packed, write, make, strides):
    _call(*_pair(make), 4, write)
    assert tuple(packed[f] for f in ("kv_sb", "kv_sh", "kv_st")) == strides


def test_c_attention_takes_shared_heads_and_tokens():
    for over in (dict(kv_sh=0), dict(kv_st=0), dict(kv_sb=0)):
        rc, need = _c_attend(**over)  # (past the checks of strides: a workspace is missing)
        assert rc == kernels.MLS_ERR_ARG and need > 0


@pytest.mark.parametrize("table", [torch.zeros(9, 64)[9:], torch.zeros(0, 32), torch.zeros(9, 128)[9:, ::2]])
def test_a_rotation_table_without_rows_is_one(packed, table):
    z = lambda *s: torch.zeros(*s, dtype=BF)
    paged_kv_append(z(4, 4, 64), z(4, 2, 64), z(4, 2, 64), z(8, 2, 16, 64), z(8, 2, 16, 64), torch.zeros(4, 3, dtype=I),
                    torch.ones(4, dtype=I), rope=table)
    assert packed["rope"] != 0 and packed["rot"] == packed["rope_ld"] == table.shape[1] and packed["rope_rows"] == 0
    assert packed["q"] != 0 and packed["q_out"] != 0


def test_c_append_rejects_rotation_without_a_table():
    a = dict.fromkeys(APPEND, 64) | dict(cu_seqlens=0, rope=0, dt=kernels.MLS_BF16, num_blocks=8, n_seqs=2, tokens=2, heads=4, kv_heads=2,
                                         block_size=16, max_blocks=3, rope_rows=0, interleaved=0)
    rc = kernels.lib().mlsx_paged_append(append_mod._ARGS.pack(*(a[f] for f in APPEND)), None)
    assert rc == kernels.MLS_ERR_ARG and b"without a table" in kernels.lib().mls_last_error()


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8, torch.uint32, torch.uint64])
def test_indexes_of_any_width(dtype):
    """What int32 cannot hold stays outside every pool and table: its low bits could be an id of one."""
    values = [0, 5, 100] + ([-1, -128] if dtype.is_signed else []) + {4: [2 ** 31 - 1], 8: [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5]}.get(dtype.itemsize, [])
    values += [2 ** 31, 2 ** 32 - 1] if dtype == torch.uint32 else [-2 ** 33 + 5, -2 ** 32] if dtype == torch.int64 else []
    got = append_mod.int32(torch.tensor(values, dtype=dtype), "block_tables", "f", (None,))
    assert got.dtype == I and got.tolist() == [min(max(v, -2 ** 31), 2 ** 31 - 1) for v in values]


def _inputs():
    z = lambda *s: torch.randn(*s)
    return dict(q=z(4, 4, 64), k=z(4, 2, 64), v=z(4, 2, 64), kp=z(8, 2, 16, 64), vp=z(8, 2, 16, 64), rope=z(9, 64), slopes=z(4))


def _run(which, a):
    tab, lens = torch.zeros(4, 3, dtype=I), torch.ones(4, dtype=I)
    if which == "append":
        return paged_kv_append(a["q"], a["k"], a["v"], a["kp"], a["vp"], tab, lens, rope=a["rope"])
    return paged_attention(a["q"], a["kp"], a["vp"], tab, lens, slopes=a["slopes"])


@pytest.mark.parametrize("which,name", [("append", n) for n in ("q", "k", "v", "kp", "vp", "rope")] + [("attend", n) for n in ("q", "kp", "vp", "slopes")])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents_and_gradients_are_refused(packed, which, name, grad_mode):
    with torch.set_grad_enabled(grad_mode):
        with forward_ad.dual_level():
            a = _inputs()
            a[name] = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
            with pytest.raises(ValueError, match="tangents"):
                _run(which, a)
            _run(which, _inputs())  # (others of the level carry none)
        if grad_mode:
            a = _inputs()
            a[name].requires_grad_()
            with pytest.raises(ValueError, match="no gradient"):
                _run(which, a)
    with pytest.raises(Exception):
        torch.func.jvp(lambda t: _run(which, {**_inputs(), name: t}), (_inputs()[name],), (_inputs()[name],))


def test_layer_refuses_inputs_that_ask_for_a_gradient(packed):
    mods = [torch.nn.Linear(128, n, bias=False) for n in (256, 128, 128)] + [torch.nn.Linear(256, 128, bias=False)]
    layer = PagedAttentionLayer(*mods, head_dim=64)
    a = _inputs()
    rest = a["kp"], a["vp"], torch.zeros(4, 3, dtype=I), torch.ones(4, dtype=I)
    x = torch.randn(4, 128)
    assert not layer(x, *rest).requires_grad
    with pytest.raises(ValueError, match="no gradient"):
        layer(x.clone().requires_grad_(), *rest)
    with torch.no_grad():
        layer(x.clone().requires_grad_(), *rest)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="tangents"):
        layer(forward_ad.make_dual(x, x), *rest)


def test_layer_made_on_the_meta_device():
    """to_empty gives its tables memory, float32 as they are."""
    with torch.device("meta"):
        mods = [torch.nn.Linear(128, n, bias=False) for n in (256, 128, 128)] + [torch.nn.Linear(256, 128, bias=False)]
        layer = PagedAttentionLayer(*mods, head_dim=64, rope=torch.zeros(9, 64), slopes=torch.zeros(4))
    layer = layer.half().to_empty(device="cpu")
    assert layer.wq.weight.dtype == torch.float16 and layer.wq.weight.device.type == "cpu"
    for t, shape in ((layer.rope, (9, 64)), (layer.slopes, (4,))):
        assert t.dtype == torch.float32 and t.device.type == "cpu" and t.shape == shape
    layer.rope.fill_(0.1)
    assert torch.equal(layer.bfloat16().rope, torch.full((9, 64), 0.1))
