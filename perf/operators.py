"""The paged serving operators as measurable cases.

Three kinds, each through a public entry point:

  append  kernels.paged_kv.paged_kv_append: new keys and values into a paged cache, rotated
          by position on the way, with the queries rotated beside them
  attend  kernels.paged_attention.paged_attention: attention of prompts, chunks and single
          tokens over the cache, grouped heads, with score options and masks
  prefix  kernels.paged_attention.shared_prefix_attention: a decode step of a batch whose
          sequences share a long prefix

A case is a dict of plain values; listed() names the fixed ones, draw(rng) makes more of the
same ranges. With own = False, run() computes the same results in elementary torch
operations, in 32 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

_PKG = str(Path(__file__).resolve().parent.parent / "mini-llm-stack_amd")

own = False

_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # The smallest call: a decode step of 8 sequences in a small fp32 model (latency counts).
        {"name": "append_fp32_s8", "kind": "append", "dtype": "fp32", "seqs": 8, "new_lo": 1, "new_hi": 1, "past_lo": 16, "past_hi": 700,
         "heads": 8, "kv_heads": 8, "dim": 64, "rot": 64, "interleaved": False, "block": 16},
        # A decode step of a full batch of a grouped-head model, half of each head rotated.
        {"name": "append_bf16_s64", "kind": "append", "dtype": "bf16", "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 1, "past_hi": 4096,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64, "interleaved": True, "block": 16},
        # Prompts of 333 to 2048 tokens admitted together.
        {"name": "append_bf16_prompts", "kind": "append", "dtype": "bf16", "seqs": 11, "new_lo": 333, "new_hi": 2048, "past_lo": 0, "past_hi": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "block": 16},
        # One sequence decoding.
        {"name": "decode_bf16_s1", "kind": "attend", "dtype": "bf16", "seqs": 1, "new_lo": 1, "new_hi": 1, "past_lo": 2047, "past_hi": 2047,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0},
        # A decode step of 40 sequences of 1 to 4096 cached tokens, scores capped.
        {"name": "decode_bf16_s40_cap", "kind": "attend", "dtype": "bf16", "seqs": 40, "new_lo": 1, "new_hi": 1, "past_lo": 1, "past_hi": 4095,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "cap": 50.0, "slopes": False, "window": 0, "prefix": 0},
        # Verification of 8 drafted tokens for 12 sequences, with a bias by distance.
        {"name": "verify_fp16_s12", "kind": "attend", "dtype": "fp16", "seqs": 12, "new_lo": 9, "new_hi": 9, "past_lo": 100, "past_hi": 2048,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 32, "cap": 0.0, "slopes": True, "window": 0, "prefix": 0},
        # Ragged chunks of long prompts in a model with a sliding window and capped scores.
        {"name": "chunk_bf16_window_cap", "kind": "attend", "dtype": "bf16", "seqs": 3, "new_lo": 200, "new_hi": 700, "past_lo": 512, "past_hi": 8192,
         "heads": 16, "kv_heads": 8, "dim": 256, "block": 16, "cap": 30.0, "slopes": False, "window": 4096, "prefix": 0},
        # Prompts of the fp32 engine, one K/V head a query head, each seeing a prefix both ways.
        {"name": "prompt_fp32_prefix_mask", "kind": "attend", "dtype": "fp32", "seqs": 5, "new_lo": 37, "new_hi": 700, "past_lo": 0, "past_hi": 0,
         "heads": 8, "kv_heads": 8, "dim": 64, "block": 16, "cap": 0.0, "slopes": False, "window": 0, "prefix": 128},
        # The largest: a long prompt in one call.
        {"name": "prompt_bf16_8192", "kind": "attend", "dtype": "bf16", "seqs": 1, "new_lo": 8192, "new_hi": 8192, "past_lo": 0, "past_hi": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0},
        # Four continuations of one system prompt.
        {"name": "prefix_bf16_s4_1000", "kind": "prefix", "dtype": "bf16", "seqs": 4, "shared": 1000, "past_lo": 0, "past_hi": 60,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "cap": 0.0, "slopes": False, "window": 0},
        # A full batch behind a long system prompt, fp16, capped.
        {"name": "prefix_fp16_s64_8192", "kind": "prefix", "dtype": "fp16", "seqs": 64, "shared": 8192, "past_lo": 1, "past_hi": 512,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "cap": 50.0, "slopes": False, "window": 0},
        # Questions about one long document.
        {"name": "prefix_bf16_s200_32768", "kind": "prefix", "dtype": "bf16", "seqs": 200, "shared": 32768, "past_lo": 10, "past_hi": 300,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 32, "cap": 0.0, "slopes": False, "window": 0},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max(-(-lo // step) * step, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "prefix", "prefix"])
    kvh = rng.choice([1, 2, 4, 8])
    c = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "kv_heads": kvh,
         "heads": min(32, kvh * rng.choice([1, 2, 4, 7, 8])), "dim": rng.choice([64, 80, 128, 128, 256]),
         "block": rng.choice([8, 16, 16, 24, 32, 64])}
    if c["heads"] % kvh:
        c["heads"] = kvh * 4
    if kind == "append":
        new = _log(rng, 1, 2048)
        c["new_lo"], c["new_hi"] = max(1, int(new * rng.uniform(0.2, 1.0))), new
        c["seqs"] = _log(rng, 1, max(1, min(128, 16384 // new)))
        past = _log(rng, 1, 4096)
        c["past_lo"], c["past_hi"] = rng.randint(0, past), past
        c["rot"] = rng.choice([c["dim"], c["dim"] // 2])
        c["interleaved"] = rng.choice([False, True])
        return c
    c["cap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
    c["slopes"] = rng.choice([False, False, True])
    if kind == "prefix":
        c["seqs"] = _log(rng, 1, 200)
        c["shared"] = _log(rng, 64, 32768 if c["dim"] <= 128 else 16384)
        c["past_lo"], c["past_hi"] = rng.randint(0, 64), _log(rng, 64, 512)
        c["window"] = rng.choice([0, 0, _log(rng, 256, 16384)])
        return c
    form = rng.choice(["decode", "decode", "verify", "prompt", "prompt"])
    if form == "decode":
        c["new_lo"], c["new_hi"], c["seqs"] = 1, 1, _log(rng, 1, 64)
        past = _log(rng, 64, 4096)
    elif form == "verify":
        n = rng.randint(2, 9)
        c["new_lo"], c["new_hi"], c["seqs"] = 1, n, _log(rng, 1, 32)
        past = _log(rng, 64, 4096)
    else:
        n = _log(rng, 32, 4096 if c["dim"] <= 128 else 2048)
        c["new_lo"], c["new_hi"] = max(1, int(n * rng.uniform(0.1, 1.0))), n
        c["seqs"] = _log(rng, 1, max(1, min(8, 4096 // n)))
        past = _log(rng, 1, 4096)
    c["past_lo"], c["past_hi"] = rng.randint(0, past), past
    c["window"] = rng.choice([0, 0, _log(rng, 128, 4096)])
    c["prefix"] = rng.choice([0, 0, _log(rng, 16, 512)])
    return c


# ---------------------------------------------------------------- inputs, from the seed alone

def _spread(lo, hi, n):
    """n whole numbers from lo to hi, even over the logarithm: the lengths of a case."""
    if n == 1:
        return [hi]
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [min(hi, max(lo, round(math.exp(a + (b - a) * i / (n - 1))) - 1)) for i in range(n)]


def _lengths(case, seed):
    """(new tokens, cached tokens before them) of every sequence, in the seed's order."""
    n = case["seqs"]
    new = _spread(case.get("new_lo", 1), case.get("new_hi", 1), n)
    past = _spread(case["past_lo"], case["past_hi"], n)
    g = torch.Generator().manual_seed(int(seed))
    o1, o2 = torch.randperm(n, generator=g).tolist(), torch.randperm(n, generator=g).tolist()
    return [new[i] for i in o1], [past[i] for i in o2]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _rotation_table(positions, rot):
    """[positions][rot] fp32: the cosines of a position's angles, then their sines (64-bit angles)."""
    j = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-2.0 * j / rot)
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def prepare(case, seed):
    c, dt, n, b = case, _DT[case["dtype"]], case["seqs"], case["block"]
    g = _gen(seed)
    new, past = _lengths(case, seed)
    total = [x + y for x, y in zip(new, past)]
    shared = -(-c.get("shared", 0) // b)
    need = [-(-t // b) for t in total]
    blocks = shared + sum(total) // b + n + 2  # as many for every order of the lengths
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(int(seed) + 1)).to(torch.int32)
    wide = max(need)
    tables = torch.zeros(n, wide, dtype=torch.int32)
    at = shared
    for s in range(n):
        tables[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    st = {"case": dict(c), "new": new, "past": past, "cu_host": cu,
          "tables": tables.cuda(), "lens": torch.tensor(total, dtype=torch.int32, device="cuda"),
          "cu": None if max(new) == 1 else torch.tensor(cu, dtype=torch.int32, device="cuda"),
          "q": _randn(g, cu[-1], c["heads"], c["dim"], dtype=dt),
          "k_pool": _randn(g, blocks, c["kv_heads"], b, c["dim"], dtype=dt),
          "v_pool": _randn(g, blocks, c["kv_heads"], b, c["dim"], dtype=dt)}
    if c["kind"] == "append":
        st["k"] = _randn(g, cu[-1], c["kv_heads"], c["dim"], dtype=dt)
        st["v"] = _randn(g, cu[-1], c["kv_heads"], c["dim"], dtype=dt)
        st["rope"] = _rotation_table(max(total), c["rot"])
        return st
    st["max_new"] = max(new)  # the program that made the batch knows it
    st["slopes"] = None
    if c["slopes"]:
        st["slopes"] = (2.0 ** (-8.0 * torch.arange(1, c["heads"] + 1, dtype=torch.float64) / c["heads"])).float().cuda()
    if c["kind"] == "prefix":
        st["shared"] = order[:shared].contiguous().cuda()
    else:
        st["prefix_lens"] = None
        if c["prefix"]:
            st["prefix_lens"] = torch.tensor([min(c["prefix"], t) for t in total], dtype=torch.int32, device="cuda")
    return st


# ---------------------------------------------------------------- one pass

def run(state):
    c = state["case"]
    if not own:
        return _PLAIN[c["kind"]](state)
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    if c["kind"] == "append":
        from kernels.paged_kv import paged_kv_append
        q = paged_kv_append(state["q"], state["k"], state["v"], state["k_pool"], state["v_pool"], state["tables"],
                            state["lens"], state["cu"], rope=state["rope"], interleaved=c["interleaved"])
        return {"q": q, "k_pool": state["k_pool"], "v_pool": state["v_pool"]}
    if c["kind"] == "attend":
        from kernels.paged_attention import paged_attention
        return paged_attention(state["q"], state["k_pool"], state["v_pool"], state["tables"], state["lens"], state["cu"],
                               max_new=state["max_new"], softcap=c["cap"], slopes=state["slopes"],
                               window=c["window"], prefix_lens=state["prefix_lens"])
    from kernels.paged_attention import shared_prefix_attention
    return shared_prefix_attention(state["q"], state["k_pool"], state["v_pool"], state["shared"], c["shared"],
                                   state["tables"], state["lens"], softcap=c["cap"], slopes=state["slopes"],
                                   window=c["window"])


def _plain_append(state):
    c = state["case"]
    lens, tables, cu = state["lens"].long(), state["tables"].long(), state["cu"]
    t = state["q"].shape[0]
    if cu is None:
        seq = torch.arange(t, device="cuda")
        pos = lens - 1
    else:
        new = (cu[1:] - cu[:-1]).long()
        seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), new, output_size=t)
        pos = torch.arange(t, device="cuda") - cu[1:].long()[seq] + lens[seq]
    half = c["rot"] // 2
    cs = state["rope"][pos]
    cos, sin = cs[:, None, :half], cs[:, None, half:]

    def turn(x):
        f = x.float()
        r, rest = f[..., :c["rot"]], f[..., c["rot"]:]
        if c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = r[..., :half], r[..., half:]
            r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([r, rest], -1).to(x.dtype)

    block, off = tables[seq, pos // c["block"]], pos % c["block"]
    state["k_pool"][block, :, off] = turn(state["k"])
    state["v_pool"][block, :, off] = state["v"]
    return {"q": turn(state["q"]), "k_pool": state["k_pool"], "v_pool": state["v_pool"]}


def _scores(x, c, slopes, dist):
    """Scaled products -> scores: the cap, then the bias by distance."""
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    if slopes is not None:
        x = x - slopes * dist.abs()
    return x


def _keys(pool, blocks, heads):
    """The pool's blocks [..., blocks] as [..., heads, tokens, dim] in 32 bits, for K/V heads heads[0] .. heads[1]."""
    x = pool[blocks, heads[0]:heads[1]]  # [..., blocks, heads, block, dim]
    x = x.movedim(-3, -4).contiguous()
    return x.reshape(*x.shape[:-3], -1, x.shape[-1]).float()


def _plain_attend(state):
    c, b = state["case"], state["case"]["block"]
    if max(state["new"]) == 1 and not c["prefix"]:
        return _plain_decode(state, None)
    kvh, group, dim = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    out = torch.empty_like(state["q"])
    for s, (new, past) in enumerate(zip(state["new"], state["past"])):
        total, row = new + past, state["cu_host"][s]
        blocks = state["tables"][s, :-(-total // b)].long()
        i = torch.arange(past, total, device="cuda")[:, None]
        j = torch.arange(total, device="cuda")[None]
        see = j <= i
        if c["prefix"]:
            see = see | (j < c["prefix"])
        if c["window"]:
            see = see & (i - j < c["window"])
        step = max(1, min(kvh, 2 ** 28 // (group * new * total)))  # K/V heads at a time
        for h in range(0, kvh, step):
            e = min(kvh, h + step)
            k = _keys(state["k_pool"], blocks, (h, e))[:, :total]
            v = _keys(state["v_pool"], blocks, (h, e))[:, :total].contiguous()
            q = state["q"][row:row + new, h * group:e * group].float()
            q = q.transpose(0, 1).reshape(e - h, group * new, dim)
            x = torch.bmm(q, k.transpose(1, 2).contiguous()).reshape(e - h, group, new, total) * dim ** -0.5
            slopes = None if state["slopes"] is None else state["slopes"][h * group:e * group].reshape(e - h, group, 1, 1)
            x = _scores(x, c, slopes, i - j)
            p = torch.softmax(x.masked_fill_(~see, float("-inf")), -1).reshape(e - h, group * new, total)
            o = torch.bmm(p, v).reshape((e - h) * group, new, dim)
            out[row:row + new, h * group:e * group] = o.transpose(0, 1).to(out.dtype)
    return out


def _plain_decode(state, shared):
    """One token a sequence: every table gathered to the longest context, with the keys of the
    shared prefix (where there is one) before them."""
    c, b = state["case"], state["case"]["block"]
    kvh, group, dim, n = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["seqs"]
    front = c["shared"] if shared is not None else 0
    lens, tables = state["lens"].long(), state["tables"].long()
    at = (front + lens - 1)[:, None]  # a sequence's position
    slopes = None if state["slopes"] is None else state["slopes"].reshape(kvh, group, 1)
    q = state["q"].reshape(n, kvh, group, dim).float()
    k, v = _keys(state["k_pool"], tables, (0, kvh)), _keys(state["v_pool"], tables, (0, kvh))
    x = torch.bmm(q.reshape(n * kvh, group, dim), k.flatten(0, 1).transpose(1, 2).contiguous())
    gap = (at - front - torch.arange(tables.shape[1] * b, device="cuda"))[:, None, None]
    x = _scores(x.reshape(n, kvh, group, -1) * dim ** -0.5, c, slopes, gap)
    see = (gap >= 0) & (gap < c["window"]) if c["window"] else gap >= 0
    x = x.masked_fill_(~see, float("-inf"))
    if shared is not None:
        kp = _keys(state["k_pool"], shared, (0, kvh))[:, :front]
        vp = _keys(state["v_pool"], shared, (0, kvh))[:, :front].contiguous()
        y = torch.bmm(q.transpose(0, 1).reshape(kvh, n * group, dim), kp.transpose(1, 2).contiguous())
        y = y.reshape(kvh, n, group, front).transpose(0, 1) * dim ** -0.5
        gap = (at - torch.arange(front, device="cuda"))[:, None, None]
        y = _scores(y, c, slopes, gap)
        if c["window"]:
            y = y.masked_fill(gap >= c["window"], float("-inf"))
        x = torch.cat([y, x], -1)
    p = torch.softmax(x, -1)
    o = torch.bmm(p[..., front:].reshape(n * kvh, group, -1), v.flatten(0, 1)).reshape(n, kvh, group, dim)
    if shared is not None:
        z = torch.bmm(p[..., :front].transpose(0, 1).reshape(kvh, n * group, front), vp)
        o = o + z.reshape(kvh, n, group, dim).transpose(0, 1)
    return o.reshape(n, kvh * group, dim).to(state["q"].dtype)


def _plain_prefix(state):
    return _plain_decode(state, state["shared"].long())


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "prefix": _plain_prefix}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    """The operators' definition, a sequence and a K/V head at a time, in 64 bits."""
    st = prepare(case, seed)
    c, b, dim, kvh = case, case["block"], case["dim"], case["kv_heads"]
    if c["kind"] == "append":
        return _exact_append(st)
    group, front = c["heads"] // kvh, c.get("shared", 0)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for s in range(c["seqs"]):
        first, count = front + st["past"][s], st["new"][s]
        end, r0 = first + count, st["cu_host"][s]
        ids = st["tables"][s, :-(-(end - front) // b)].long()
        cols = torch.arange(end, device="cuda", dtype=torch.float64)
        for h in range(kvh):
            parts = []
            for pool in (st["k_pool"], st["v_pool"]):
                mine = pool[ids, h].flatten(0, 1)[:end - front]
                if front:
                    mine = torch.cat([pool[st["shared"].long(), h].flatten(0, 1)[:front], mine])
                parts.append(mine.double())
            keys, values = parts
            for lo in range(0, count, 1024):  # query rows in pieces that bound the score matrix
                hi = min(count, lo + 1024)
                at = torch.arange(first + lo, first + hi, device="cuda", dtype=torch.float64)
                gap = at[:, None] - cols[None, :]
                hidden = gap < 0
                if c.get("prefix", 0):
                    hidden &= (cols >= c["prefix"])[None, :]
                if c["window"]:
                    hidden |= gap >= c["window"]
                for a in range(group):
                    head = h * group + a
                    z = torch.mm(st["q"][r0 + lo:r0 + hi, head].double(), keys.t()) / math.sqrt(dim)
                    if c["cap"]:
                        z = torch.tanh(z / c["cap"]) * c["cap"]
                    if st["slopes"] is not None:
                        z = z - st["slopes"][head].double() * gap.abs()
                    z[hidden] = float("-inf")
                    w = torch.exp(z - z.max(dim=1, keepdim=True).values)
                    out[r0 + lo:r0 + hi, head] = torch.mm(w, values) / w.sum(dim=1, keepdim=True)
    return out


def _exact_append(st):
    c = st["case"]
    half, b = c["rot"] // 2, c["block"]
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    q = st["q"].double()
    k = st["k"].double()
    kp, vp = st["k_pool"].double(), st["v_pool"].double()
    even = torch.arange(half, device="cuda") * 2 if c["interleaved"] else torch.arange(half, device="cuda")
    odd = even + (1 if c["interleaved"] else half)
    for s in range(c["seqs"]):
        r0, r1 = st["cu_host"][s], st["cu_host"][s + 1]
        at = torch.arange(st["past"][s], st["past"][s] + st["new"][s], device="cuda")
        turn = torch.polar(torch.ones(r1 - r0, half, dtype=torch.float64, device="cuda"), at.double()[:, None] * freq)
        for x in (q, k):
            z = torch.complex(x[r0:r1][..., even], x[r0:r1][..., odd]) * turn[:, None]
            x[r0:r1, :, even] = z.real
            x[r0:r1, :, odd] = z.imag
        slot = st["tables"][s].long()[at // b]
        kp[slot, :, at % b] = k[r0:r1]
        vp[slot, :, at % b] = st["v"][r0:r1].double()
    return {"q": q, "k_pool": kp, "v_pool": vp}


# ---------------------------------------------------------------- what a pass cannot do without

def _visible(first, count, window, prefix, end):
    """Keys that the tokens at first .. first + count see, summed, and the keys that any of them sees."""
    pairs = 0
    for i in range(first, first + count):
        hi = max(i + 1, min(prefix, end))
        lo = max(0, i - window + 1) if window else 0
        pairs += hi - lo
    lo = max(0, first - window + 1) if window else 0
    return pairs, max(first + count, min(prefix, end)) - lo


def work(case):
    c, size = case, _BYTES[case["dtype"]]
    new, past = _lengths(case, 0)
    rows = sum(new)
    if c["kind"] == "append":
        per = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": 2 * rows * per * size + rows * c["rot"] * 4,
                "flops": 3 * rows * (c["heads"] + c["kv_heads"]) * c["rot"]}
    front = c.get("shared", 0)
    pairs = keys = 0
    for x, y in zip(sorted(new), sorted(past)):
        p, k = _visible(front + y, x, c["window"], c.get("prefix", 0), front + y + x)
        pairs += p
        keys += min(k, x + y)
    keys += min(front, max(0, c["window"] or front)) if front else 0
    return {"bytes": (2 * keys * c["kv_heads"] + 2 * rows * c["heads"]) * c["dim"] * size,
            "flops": 4 * pairs * c["heads"] * c["dim"]}
