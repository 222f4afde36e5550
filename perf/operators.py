"""Cases that time the rotary, paged-cache and paged-attention operators.

``run`` computes one pass of an operator: in its plain form (elementary torch
operations in fp32, angles in fp64) where ``own`` is false, through the
package's public operators where it is true.  ``exact`` gives the same outputs
from the definitions in fp64.

The operators, for a sequence b of ``q_len`` new tokens whose cache holds
``kv_len`` tokens with the new ones counted (token i sits at position
``kv_len - q_len + i``; key j of sequence b is row ``j % page`` of page
``block_table[b, j // page]``):

* rotary:     (a, b) -> (a cos t - b sin t, b cos t + a sin t) for the pairs of
              the first R of D channels, t = position * inv_freq, each
              frequency's position taken from its own axis;
* append:     rotates new keys (and queries), writes keys and values to their
              places in the cache;
* attention:  softmax(q k^T * scale) v of each new token over the keys up to its
              own position (or over all of the sequence's), heads in groups
              that share a key/value head.
"""

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PAGES = (16, 32, 64, 128)


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _rotary(name, kind, B, H, S, D, R, axes=1, packed=False, interleaved=False, inverse=False,
            far=8192, base=10000.0):
    return {"name": name, "op": "rotary", "type": kind, "B": B, "H": H, "S": S, "D": D, "R": R,
            "axes": axes, "packed": packed, "interleaved": interleaved, "inverse": inverse,
            "far": far, "base": base}


def _append(name, kind, B, q_max, kv_max, Hq, Hkv, D, R, page, axes=1, interleaved=False, mix=1,
            base=10000.0):
    return {"name": name, "op": "append", "type": kind, "B": B, "q_max": q_max, "kv_max": kv_max,
            "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "page": page, "axes": axes,
            "interleaved": interleaved, "mix": mix, "base": base}


def _attention(name, kind, B, q_max, kv_max, Hq, Hkv, D, page, causal=True, mix=1):
    return {"name": name, "op": "attention", "type": kind, "B": B, "q_max": q_max,
            "kv_max": kv_max, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "causal": causal,
            "mix": mix}


def listed():
    return [
        # queries of one generation step of eight sequences: a pure latency case
        _rotary("rotary_step", "bf16", 8, 16, 1, 64, 64, far=4096),
        # the gradient's direction on the [B, H, S, D] layout, odd length, neighbouring pairs
        _rotary("rotary_inverse_odd", "fp32", 2, 16, 2047, 64, 64, interleaved=True, inverse=True),
        # rows of a long prompt with video: time, height and width positions
        _rotary("rotary_video", "bf16", 1, 32, 16384, 128, 128, axes=3, packed=True, far=131072,
                base=500000.0),
        # one generation step of 32 sequences: rotate q and k, store k and v
        _append("append_step", "bf16", 32, 1, 4096, 32, 8, 128, 128, 16),
        # ragged chunks of five prompts, half of each head rotated
        _append("append_chunks", "fp16", 5, 4096, 16384, 16, 16, 128, 64, 64, mix=3),
        # one short sequence's next token
        _attention("step_one", "bf16", 1, 1, 500, 16, 16, 64, 16),
        # a generation step of 32 ragged sequences, four query heads to a key head
        _attention("step_batch", "bf16", 32, 1, 8192, 32, 8, 128, 16, mix=2),
        # a few very long contexts, where the work has to be split along the keys
        _attention("step_long", "fp16", 3, 1, 131072, 32, 4, 128, 64, mix=5),
        # a short odd chunk behind a medium cache
        _attention("chunk_short", "fp16", 1, 37, 1061, 16, 16, 64, 32),
        # chunks of prompts and single tokens in one batch
        _attention("chunk_mixed", "bf16", 9, 700, 6000, 32, 8, 128, 16, mix=4),
        # a chunk of a long prompt behind the chunks before it
        _attention("chunk_long", "bf16", 1, 512, 32768, 32, 8, 128, 64),
        # a whole prompt of 8192 tokens and 32 heads
        _attention("prompt", "bf16", 1, 8192, 8192, 32, 32, 128, 128),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    group = rng.choice((1, 2, 3, 4, 5, 6, 7, 8, 12, 16))
    kv = rng.choice((1, 2, 3, 4, 8, 16))
    while group * kv > 64:
        kv = max(1, kv // 2)
    return group * kv, kv


def draw(rng):
    op = rng.choice(("rotary", "append", "attention", "attention", "attention"))
    half = rng.choice(("bf16", "fp16"))
    if op == "rotary":
        kind = rng.choice(("bf16", "fp16", "fp32"))
        packed = rng.random() < 0.5
        D = rng.choice((32, 64, 80, 96, 128, 192, 256))
        R = min(D, rng.choice((16, 32, 64, 96, 128, 256)))
        H = rng.choice((1, 2, 5, 8, 16, 24, 32, 48))
        B = 1 if packed else _spread(rng, 1, 16)
        S = _spread(rng, 1, max(1, 16384 * 4096 // (B * H * D)))
        axes = rng.choice((1, 1, 2, 3, 4))
        case = _rotary("", kind, B, H, S, D, R, axes, packed, rng.random() < 0.3,
                       rng.random() < 0.3, _spread(rng, 64, 1 << 20),
                       rng.choice((10000.0, 500000.0)))
    elif op == "append":
        Hq, Hkv = _heads(rng)
        D = rng.choice((64, 80, 96, 128))
        R = min(D, rng.choice((32, 64, 96, 128)))
        B = _spread(rng, 1, 64)
        q_max = 1 if rng.random() < 0.4 else _spread(rng, 2, max(2, 16384 // B))
        kv_max = _spread(rng, max(q_max, 16), max(q_max, 16, (1 << 27) // (B * Hkv * D)))
        case = _append("", half, B, q_max, kv_max, Hq, Hkv, D, R, rng.choice(PAGES),
                       rng.choice((1, 1, 3)), rng.random() < 0.3, rng.randrange(1 << 16),
                       rng.choice((10000.0, 500000.0)))
    else:
        Hq, Hkv = _heads(rng)
        D = rng.choice((32, 64, 64, 80, 96, 128, 128, 128))
        B = _spread(rng, 1, 48)
        q_max = 1 if rng.random() < 0.4 else _spread(rng, 2, 2048)
        while B > 1 and B * Hq * q_max * max(q_max, 16) > 1 << 29:
            B -= 1
        kv_top = min(131072, (1 << 29) // (B * Hq * q_max), (1 << 27) // (B * Hkv * D))
        kv_max = _spread(rng, max(q_max, 16), max(q_max, 16, kv_top))
        case = _attention("", half, B, q_max, kv_max, Hq, Hkv, D, rng.choice(PAGES),
                          rng.random() < 0.85, rng.randrange(1 << 16))
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """The batch's (q_len, kv_len) pairs: by the case alone, the longest of each among them."""
    rng = random.Random(case["mix"])
    pairs = []
    for b in range(case["B"]):
        q = case["q_max"]
        if b and q > 1:
            q = 1 if rng.random() < 0.4 else rng.randint(1, q)
        kv = case["kv_max"] if b == 0 else rng.randint(max(q, case["kv_max"] // 4), case["kv_max"])
        pairs.append((q, kv))
    rng.shuffle(pairs)
    return pairs


def _sections(R, axes):
    """How many of the R/2 frequencies each axis has (the last axes alike, the rest to the first)."""
    if axes == 1:
        return None
    each = R // 2 * 3 // (4 * axes - 4) if axes > 2 else R // 4
    return (R // 2 - each * (axes - 1),) + (each,) * (axes - 1)


def _frequencies(case):
    i = torch.arange(0, case["R"], 2, dtype=torch.float64)
    return (case["base"] ** (-i / case["R"])).to(torch.float32).to("cuda")


def _axis_positions(gen, axes, S, far):
    """Axis 0 counts on from some start, the others are places in a frame."""
    start = int(torch.randint(0, max(1, far - S), (1,), generator=gen, device="cuda"))
    first = torch.arange(start, start + S, device="cuda").unsqueeze(0)
    rest = torch.randint(0, min(far, 1024), (axes - 1, S), generator=gen, device="cuda")
    return torch.cat([first, rest])


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    kind = TYPES[case["type"]]
    state = {"case": case}
    if case["op"] == "rotary":
        shape = ((case["S"], case["H"], case["D"]) if case["packed"]
                 else (case["B"], case["H"], case["S"], case["D"]))
        state["x"] = torch.randn(shape, generator=gen, device="cuda").to(kind)
        positions = _axis_positions(gen, case["axes"], case["S"], case["far"])
        state["positions"] = (positions if case["axes"] > 1 else positions[0]).to(torch.int32)
        state["inv_freq"] = _frequencies(case)
        state["sections"] = _sections(case["R"], case["axes"])
        return state

    pairs = _lengths(case)
    B, page, Hq, Hkv, D = case["B"], case["page"], case["Hq"], case["Hkv"], case["D"]
    T = sum(q for q, _ in pairs)
    starts = [0]
    for q, _ in pairs:
        starts.append(starts[-1] + q)
    used = [-(-kv // page) for _, kv in pairs]
    total = sum(used) + 8
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((B, max(used)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    state["block_table"] = table
    state["cu_seqlens"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    state["kv_lens"] = torch.tensor([kv for _, kv in pairs], dtype=torch.int32, device="cuda")
    state["max_q_len"] = max(q for q, _ in pairs)
    state["max_kv_len"] = max(kv for _, kv in pairs)
    for name in ("k_cache", "v_cache"):
        state[name] = torch.randn((total, page, Hkv, D), generator=gen, device="cuda",
                                  dtype=kind)
    if case["op"] == "append":
        # one projection's rows: queries, keys and values of a token side by side
        rows = torch.randn((T, (Hq + 2 * Hkv) * D), generator=gen, device="cuda").to(kind)
        q, k, v = rows.split([Hq * D, Hkv * D, Hkv * D], dim=1)
        state["q"], state["k"], state["v"] = (t.unflatten(1, (-1, D)) for t in (q, k, v))
        state["inv_freq"] = _frequencies(case)
        state["sections"] = _sections(case["R"], case["axes"])
        state["positions"] = None
        if case["axes"] > 1:
            state["positions"] = _axis_positions(gen, case["axes"], T,
                                                 case["kv_max"]).to(torch.int32)
    else:
        state["q"] = torch.randn((T, Hq, D), generator=gen, device="cuda").to(kind)
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    return {"rotary": _plain_rotary, "append": _plain_append,
            "attention": _plain_attention}[case["op"]](state, case)


def _run_own(state, case):
    import cs348k_fast_attention_grammar_b200 as fa

    if case["op"] == "rotary":
        return fa.rotary(state["x"], state["positions"], state["inv_freq"],
                         sections=state["sections"], interleaved=case["interleaved"],
                         inverse=case["inverse"])
    if case["op"] == "append":
        q = fa.paged_kv_append(state["k"], state["v"], state["k_cache"], state["v_cache"],
                               state["block_table"], state["kv_lens"],
                               cu_seqlens=state["cu_seqlens"], q=state["q"],
                               inv_freq=state["inv_freq"], positions=state["positions"],
                               sections=state["sections"], interleaved=case["interleaved"])
        return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    return fa.paged_attention(state["q"], state["k_cache"], state["v_cache"],
                              state["block_table"], state["kv_lens"],
                              cu_seqlens=state["cu_seqlens"], max_q_len=state["max_q_len"],
                              causal=case["causal"])


def _turn(x, angle, R, interleaved, inverse):
    """Rotates the first R channels of fp32 x by fp64 angles [..., R/2], rounded by the caller."""
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    sin = -sin if inverse else sin
    r = x[..., :R]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :R // 2], r[..., R // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, x[..., R:]], -1)


def _angles(positions, inv_freq, sections):
    """fp64 angles [..., R/2] of positions [...], or [axes, ...] where there are sections."""
    f = inv_freq.double()
    if sections is None:
        return positions.double().unsqueeze(-1) * f
    count = torch.tensor(sections, device=f.device)
    axis = torch.repeat_interleave(torch.arange(len(sections), device=f.device), count,
                                   output_size=f.numel())
    return positions.double()[axis].movedim(0, -1) * f


def _plain_rotary(state, case):
    angle = _angles(state["positions"], state["inv_freq"], state["sections"])
    if case["packed"]:
        angle = angle.unsqueeze(1)
    x = state["x"]
    return _turn(x.float(), angle, case["R"], case["interleaved"], case["inverse"]).to(x.dtype)


def _places(state, T):
    """Sequence and cache position of each new token."""
    cu = state["cu_seqlens"].long()
    row = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu[1:], row, right=True)
    return b, row - cu[1:][b] + state["kv_lens"].long()[b]


def _plain_append(state, case):
    T, page = state["k"].shape[0], case["page"]
    b, at = _places(state, T)
    positions = at if state["positions"] is None else state["positions"]
    angle = _angles(positions, state["inv_freq"], state["sections"]).unsqueeze(1)
    q, k = (_turn(state[n].float(), angle, case["R"], case["interleaved"], False).to(
        state[n].dtype) for n in ("q", "k"))
    place = state["block_table"].long()[b, at // page] * page + at % page
    state["k_cache"].flatten(0, 1)[place] = k
    state["v_cache"].flatten(0, 1)[place] = state["v"]
    return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


def _plain_attention(state, case):
    q, Hkv, D = state["q"], case["Hkv"], case["D"]
    T, B, qm, km = q.shape[0], case["B"], state["max_q_len"], state["max_kv_len"]
    group = case["Hq"] // Hkv
    cu, lens = state["cu_seqlens"].long(), state["kv_lens"].long()
    table = state["block_table"].long().clamp(min=0)
    # [B, Hkv, keys, D] and [B, Hkv, group * queries, D], padded to the longest
    k, v = (state[n][table].flatten(1, 2)[:, :km].float().transpose(1, 2)
            for n in ("k_cache", "v_cache"))
    step = torch.arange(qm, device=q.device)
    rows = (cu[:-1, None] + step).clamp(max=T - 1)
    qp = q[rows].float().unflatten(2, (Hkv, group)).permute(0, 2, 3, 1, 4)
    s = qp.flatten(2, 3) @ k.transpose(2, 3) * (1.0 / math.sqrt(D))
    s = s.unflatten(2, (group, qm))
    key = torch.arange(km, device=q.device)
    last = lens[:, None] - 1
    if case["causal"]:
        last = last - (cu[1:] - cu[:-1])[:, None] + 1 + step
    seen = (key <= last.unsqueeze(-1)) & (key < lens[:, None, None])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp_(s.sub_(torch.where(m == -math.inf, 0.0, m)))
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (group, qm))
    o = torch.where(total > 0, o / total, 0.0)
    b, at = _places(state, T)
    i = at - lens[b] + (cu[1:] - cu[:-1])[b]
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3)[b, i].to(q.dtype)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = TYPES[case["type"]].itemsize
    if case["op"] == "rotary":
        rows = case["B"] * case["S"]
        n = rows * case["H"]
        return {"bytes": 2 * n * case["D"] * size + case["S"] * case["axes"] * 4 + case["R"] * 2,
                "flops": 3 * n * case["R"]}
    pairs = _lengths(case)
    T = sum(q for q, _ in pairs)
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    if case["op"] == "append":
        return {"bytes": 2 * T * (Hq + 2 * Hkv) * D * size + 4 * T,
                "flops": 3 * T * (Hq + Hkv) * case["R"]}
    keys = sum(kv for _, kv in pairs)
    if case["causal"]:
        seen = sum(q * (kv - q) + q * (q + 1) // 2 for q, kv in pairs)
    else:
        seen = sum(q * kv for q, kv in pairs)
    return {"bytes": 2 * keys * Hkv * D * size + 2 * T * Hq * D * size
            + 4 * sum(-(-kv // case["page"]) for _, kv in pairs),
            "flops": 4 * seen * Hq * D}


# ---------------------------------------------------------------------------
# The definitions in fp64
# ---------------------------------------------------------------------------
def _exact_rotation(x, positions, case, sections, inverse):
    """x [rows, heads, D] with positions [axes, rows]: one plane at a time as a complex product."""
    R = case["R"]
    y = x.double().clone()
    freq = [float(f) for f in _frequencies(case).cpu()]
    ends = [sum((sections or (R // 2,))[:a + 1]) for a in range(len(sections or (1,)))]
    for i, f in enumerate(freq):
        axis = next(a for a, end in enumerate(ends) if i < end)
        t = positions[axis].double() * f
        spin = torch.polar(torch.ones_like(t), -t if inverse else t)[:, None]
        at = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + R // 2)
        z = torch.complex(x[..., at[0]].double(), x[..., at[1]].double()) * spin
        y[..., at[0]], y[..., at[1]] = z.real, z.imag
    return y


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        x = state["x"]
        positions = state["positions"].reshape(case["axes"], -1)
        if case["packed"]:
            return _exact_rotation(x, positions, case, state["sections"], case["inverse"])
        rows = x.permute(0, 2, 1, 3).flatten(0, 1)
        y = _exact_rotation(rows, positions.repeat(1, case["B"]), case, state["sections"],
                            case["inverse"])
        return y.unflatten(0, (case["B"], case["S"])).permute(0, 2, 1, 3).contiguous()
    pairs, page = _lengths(case), case["page"]
    if case["op"] == "append":
        k_cache, v_cache = state["k_cache"].double(), state["v_cache"].double()
        positions = state["positions"]
        if positions is None:
            positions = torch.cat([torch.arange(kv - q, kv) for q, kv in pairs])[None].to("cuda")
        q, k = (_exact_rotation(state[n], positions, case, state["sections"], False)
                for n in ("q", "k"))
        table, row = state["block_table"].cpu(), 0
        for b, (n, kv) in enumerate(pairs):
            places = [int(table[b, j // page]) * page + j % page for j in range(kv - n, kv)]
            places = torch.tensor(places, device="cuda")
            k_cache.view(-1, *k.shape[1:])[places] = k[row:row + n]
            v_cache.view(-1, *k.shape[1:])[places] = state["v"][row:row + n].double()
            row += n
        return {"q": q, "k_cache": k_cache, "v_cache": v_cache}
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    group, row = case["Hq"] // case["Hkv"], 0
    for b, (n, kv) in enumerate(pairs):
        pages = state["block_table"][b, :-(-kv // page)].long()
        later = torch.arange(kv, device="cuda")[None] > torch.arange(kv - n, kv,
                                                                     device="cuda")[:, None]
        for h in range(case["Hkv"]):
            k, v = (state[c][pages][:, :, h].reshape(-1, case["D"])[:kv].double()
                    for c in ("k_cache", "v_cache"))
            for g in range(h * group, (h + 1) * group):
                s = state["q"][row:row + n, g].double() @ k.T / math.sqrt(case["D"])
                if case["causal"]:
                    s = s.masked_fill(later, -math.inf)
                out[row:row + n, g] = torch.softmax(s, -1) @ v
        row += n
    return out
