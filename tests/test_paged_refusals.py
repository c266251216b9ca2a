"""What paged_kv_append, paged_attention and shared_prefix_attention refuse, on the host: the wrappers' checks on CPU
tensors, which come before any kernel, and the C entries' with addresses that nothing reads."""

from __future__ import annotations

import struct

import pytest
import torch

import kernels
from kernels.paged_attention import _ARGS, paged_attention, shared_prefix_attention
from kernels.paged_kv import _ARGS as _APPEND, paged_kv_append

I = torch.int32


def _in(T=4, n=4, Hq=4, Hkv=2, D=64, bs=16, dtype=torch.bfloat16):
    z = lambda *s: torch.zeros(*s, dtype=dtype)
    return dict(q=z(T, Hq, D), k=z(T, Hkv, D), v=z(T, Hkv, D), kp=z(8, Hkv, bs, D), vp=z(8, Hkv, bs, D),
                tab=torch.zeros(n, 3, dtype=I), lens=torch.ones(n, dtype=I), cu=None, rope=None)


def _append(**over):
    a = {**_in(), **over}
    return paged_kv_append(a["q"], a["k"], a["v"], a["kp"], a["vp"], a["tab"], a["lens"], a["cu"], rope=a["rope"])


def _attend(opts=None, **over):
    a = {**_in(), **over}
    return paged_attention(a["q"], a["kp"], a["vp"], a["tab"], a["lens"], a["cu"], **(opts or {}))


BF, FP = torch.bfloat16, torch.float32
SHARED = [
    (dict(kp=torch.zeros(8, 2, 16, dtype=BF)), ValueError), (dict(vp=torch.zeros(8, 2, 16, 32, dtype=BF)), ValueError),
    (dict(vp=torch.zeros(8, 2, 16, 64)), ValueError), (dict(vp=torch.zeros(8, 16, 2, 64, dtype=BF).transpose(1, 2)), ValueError),
    (dict(kp=torch.zeros(8, 2, 64, 16, dtype=BF).transpose(2, 3), vp=torch.zeros(8, 2, 64, 16, dtype=BF).transpose(2, 3)), ValueError),
    (dict(kp=torch.zeros(8, 2, 0, 64, dtype=BF), vp=torch.zeros(8, 2, 0, 64, dtype=BF)), ValueError),
    (dict(q=torch.zeros(4, 4, 64)), TypeError), (dict(q=torch.zeros(4, 4, 32, dtype=BF)), ValueError),
    (dict(tab=torch.zeros(3, 3, dtype=I)), ValueError), (dict(tab=torch.zeros(4, dtype=I)), ValueError),
    (dict(tab=torch.zeros(4, 3)), TypeError), (dict(lens=torch.ones(4)), TypeError), (dict(lens=torch.ones(4, 1, dtype=I)), ValueError),
    (dict(lens=torch.ones(3, dtype=I), tab=torch.zeros(3, 3, dtype=I)), ValueError), (dict(cu=torch.zeros(4, dtype=I)), ValueError),
    (dict(cu=torch.zeros(5)), TypeError), ({}, TypeError),  # (the last: CPU tensors)
]


@pytest.mark.parametrize("over,error", SHARED + [
    (dict(v=torch.zeros(4, 2, 32, dtype=BF)), ValueError), (dict(k=torch.zeros(4, 3, 64, dtype=BF), v=torch.zeros(4, 3, 64, dtype=BF)), ValueError),
    (dict(k=torch.zeros(4, 2, 64)), TypeError), (dict(q=torch.zeros(3, 4, 64, dtype=BF)), ValueError),
    (dict(rope=torch.zeros(9, 63)), ValueError), (dict(rope=torch.zeros(9, 66)), ValueError), (dict(rope=torch.zeros(9, 64, dtype=BF)), ValueError),
    (dict(rope=torch.zeros(64)), ValueError), (dict(k=torch.zeros(4, 2, 64, dtype=BF, requires_grad=True)), ValueError),
])
def test_append_refuses(over, error):
    with pytest.raises(error):
        _append(**over)


@pytest.mark.parametrize("over,error", SHARED + [
    (dict(q=torch.zeros(4, 3, 64, dtype=BF)), ValueError), (dict(q=torch.zeros(4, 64, dtype=BF)), ValueError),
    (dict(q=torch.zeros(4, 4, 64, dtype=BF, requires_grad=True)), ValueError),
])
def test_attention_refuses(over, error):
    with pytest.raises(error):
        _attend(**over)


@pytest.mark.parametrize("opts", [dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(window=-1),
                                  dict(max_new=-1), dict(slopes=torch.zeros(2)), dict(slopes=torch.zeros(4, dtype=BF)),
                                  dict(prefix_lens=torch.zeros(3, dtype=I))])
def test_attention_refuses_options(opts):
    with pytest.raises(ValueError):
        _attend(opts)


@pytest.mark.parametrize("blocks,length", [(3, 49), (3, -1), (0, 1)])
def test_shared_prefix_refuses(blocks, length):
    a = _in()
    with pytest.raises(ValueError):
        shared_prefix_attention(a["q"], a["kp"], a["vp"], torch.zeros(blocks, dtype=I), length, a["tab"], a["lens"])


ATTEND = ["q", "k_pool", "v_pool", "block_tables", "context_lens", "cu_seqlens", "prefix_lens", "prefix_blocks", "slopes", "out", "dt",
          "q_st", "q_sh", "o_st", "o_sh", "kv_sb", "kv_sh", "kv_st", "bt_ss", "num_blocks", "n_seqs", "tokens", "kv_heads", "group",
          "head_dim", "block_size", "max_blocks", "window", "prefix_len", "prefix_count", "max_new", "scale", "softcap"]
APPEND = ["q", "k", "v", "k_pool", "v_pool", "q_out", "block_tables", "context_lens", "cu_seqlens", "rope", "dt", "q_st", "q_sh", "k_st",
          "k_sh", "v_st", "v_sh", "kv_sb", "kv_sh", "kv_st", "bt_ss", "rope_ld", "num_blocks", "n_seqs", "tokens", "heads", "kv_heads",
          "head_dim", "block_size", "max_blocks", "rope_rows", "rot", "interleaved"]


def _c_attend(ws=0, **over):
    a = dict(q=64, k_pool=64, v_pool=64, block_tables=64, context_lens=64, cu_seqlens=0, prefix_lens=0, prefix_blocks=0, slopes=0,
             out=64, dt=kernels.MLS_BF16, q_st=256, q_sh=64, o_st=256, o_sh=64, kv_sb=2048, kv_sh=1024, kv_st=64, bt_ss=300,
             num_blocks=8, n_seqs=2, tokens=2, kv_heads=2, group=2, head_dim=64, block_size=16, max_blocks=300, window=0, prefix_len=0,
             prefix_count=0, max_new=0, scale=0.125, softcap=0.0)
    assert not set(over) - set(a)
    packed = _ARGS.pack(*({**a, **over}[k] for k in ATTEND))
    return kernels.lib().mlsx_paged_attention(packed, ws or None, 1 if ws else 0, None), kernels.lib().mlsx_paged_attention_ws(packed)


@pytest.mark.parametrize("over", [dict(q=0), dict(k_pool=0), dict(out=0), dict(context_lens=0), dict(block_tables=0), dict(dt=3),
                                  dict(head_dim=-1), dict(block_size=0), dict(tokens=3), dict(max_blocks=-1), dict(window=-1), dict(q_sh=63),
                                  dict(kv_st=63), dict(kv_sb=-1), dict(softcap=-1.0), dict(softcap=float("nan")), dict(o_st=100),
                                  dict(prefix_blocks=64, cu_seqlens=64, prefix_len=4, prefix_count=1)])
def test_c_attention_rejects(over):
    rc, need = _c_attend(**over)
    assert rc == kernels.MLS_ERR_ARG and need == 0 and b"mlsx_paged_attention" in kernels.lib().mls_last_error()


def test_c_attention_limits():
    assert _c_attend(head_dim=257, q_sh=257, kv_st=257, q_st=1028, o_st=1028, o_sh=257)[0] == kernels.MLS_ERR_UNSUPPORTED
    assert _c_attend(tokens=1 << 30, n_seqs=1 << 30)[0] == kernels.MLS_ERR_UNSUPPORTED
    rc, need = _c_attend()  # 4800 tokens in pieces: a workspace is needed
    assert rc == kernels.MLS_ERR_ARG and need > 0
    assert _c_attend(ws=64)[0] == kernels.MLS_ERR_ARG  # too small
    assert _c_attend(n_seqs=0, tokens=0) == (0, 0)
    assert kernels.lib().mlsx_paged_attention(None, None, 0, None) == kernels.MLS_ERR_ARG
    assert kernels.lib().mlsx_paged_attention_ws(None) == 0


@pytest.mark.parametrize("over", [dict(k=0), dict(v=0), dict(k_pool=0), dict(context_lens=0), dict(q_out=0), dict(dt=9), dict(tokens=3),
                                  dict(rot=3), dict(rot=66), dict(rope_ld=10), dict(kv_st=9), dict(k_st=-1), dict(block_size=0),
                                  dict(rope_rows=-1)])
def test_c_append_rejects(over):
    a = dict(q=64, k=64, v=64, k_pool=64, v_pool=64, q_out=64, block_tables=64, context_lens=64, cu_seqlens=0, rope=64,
             dt=kernels.MLS_BF16, q_st=256, q_sh=64, k_st=128, k_sh=64, v_st=128, v_sh=64, kv_sb=2048, kv_sh=1024, kv_st=64, bt_ss=3,
             rope_ld=64, num_blocks=8, n_seqs=2, tokens=2, heads=4, kv_heads=2, head_dim=64, block_size=16, max_blocks=3, rope_rows=9,
             rot=64, interleaved=0)
    assert not set(over) - set(a)
    rc = kernels.lib().mlsx_paged_append(_APPEND.pack(*({**a, **over}[k] for k in APPEND)), None)
    assert rc == kernels.MLS_ERR_ARG and b"mlsx_paged_append" in kernels.lib().mls_last_error()


def test_argument_structs_have_the_headers_fields():
    """The packed structs list the header's fields in its order, 8 bytes each."""
    from conftest import ROOT
    import re
    text = (ROOT / "include" / "mls_ext.h").read_text()
    for name, fields, packed in (("mlsx_paged_attention_args", ATTEND, _ARGS), ("mlsx_paged_append_args", APPEND, _APPEND)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        got = [w.strip(" *\n") for line in body.split(";") for w in re.sub(r"^\s*(const\s+)?(void|int32_t|int64_t|float|double)\b", "", line.strip("\n ")).split(",")]
        assert [g for g in got if g] == fields and packed.size == 8 * len(fields) and struct.calcsize("P") == 8
