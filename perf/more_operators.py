"""Operators of a serving loop around a compressed cache, as timed cases with their plain forms.

``op`` names what one pass does:

* ``rotate``  queries and keys turned by their positions, and the keys and values appended: ``step`` a few tokens of
  every sequence of a batch into the dense tail (and the cache taken back to its length), ``prompt`` a prompt into a
  new cache, with the history handed back decompressed, as the prompt's attention reads it;
* ``shared``  one decode step's attention of a batch whose sequences share a prefix that is stored once, each with
  tokens of its own behind it;
* ``bounds``  the smallest and the largest of every key component over each page;
* ``select``  one decode step's attention over the pages whose bounds allow the largest scores, the first and the last
  pages and the dense tail.

With ``own`` false ``run`` computes them in elementary torch operations in 32 bits (64 for the rotation, whose keys are
rounded to codes, and for the scores that pages are chosen by); with ``own`` true it makes the calls of this
repository's package.
"""

import json
import math
import random

import numpy as np
import torch

own = False

PAGE, DIM, PAIRS = 64, 128, 64

# int8 log radii, level-1 bits, deep bits, split: the configuration's defaults, the layout of make_turbo_caches, and
# other widths that the configuration takes.
LAYOUTS = {
    "default": (False, 4, 4, 64),
    "fast": (True, 4, 8, 0),
    "deep2": (False, 4, 2, 64),
    "l1_8bit": (False, 8, 4, 32),
    "odd_split": (True, 4, 2, 46),
    "int8_angles4": (True, 4, 4, 64),
}

# (query heads, kv heads) of the configurations, the tests and the benchmark.
HEADS = [(32, 8), (64, 8), (32, 32), (8, 8), (28, 4), (40, 8), (4, 1), (8, 1), (16, 4), (24, 2), (40, 2), (8, 2)]


def listed():
    return [
        # One token of a chat, where latency counts.
        {"name": "rotate_1", "op": "rotate", "kind": "step", "layout": "fast", "dtype": "float16", "tables": "float16",
         "interleaved": False, "batch": 1, "hq": 32, "hkv": 8, "tokens": 300, "new": 1},
        # A serving batch's step, in the types of a bfloat16 model with its tables kept in 32 bits.
        {"name": "rotate_batch", "op": "rotate", "kind": "step", "layout": "default", "dtype": "bfloat16",
         "tables": "float32", "interleaved": False, "batch": 48, "hq": 64, "hkv": 8, "tokens": 80, "new": 1},
        # An ordinary prompt into a new cache.
        {"name": "rotate_4k", "op": "rotate", "kind": "prompt", "layout": "fast", "dtype": "bfloat16",
         "tables": "bfloat16", "interleaved": False, "batch": 1, "hq": 32, "hkv": 8, "tokens": 0, "new": 4100},
        # A long document, pairs of neighbours turned, its end inside a page.
        {"name": "rotate_32k", "op": "rotate", "kind": "prompt", "layout": "default", "dtype": "float16",
         "tables": "float32", "interleaved": True, "batch": 1, "hq": 32, "hkv": 8, "tokens": 0, "new": 32773},
        # A few samples of one question: a short common prompt, short answers.
        {"name": "shared_1k", "op": "shared", "layout": "default", "batch": 4, "hq": 32, "hkv": 8, "prefix": 1000,
         "tokens": 50},
        # A serving batch behind a long common document, some hundred tokens each.
        {"name": "shared_32k", "op": "shared", "layout": "default", "batch": 32, "hq": 32, "hkv": 8, "prefix": 32805,
         "tokens": 300},
        # Many short requests behind one system prompt, eight query heads a group.
        {"name": "shared_wide", "op": "shared", "layout": "fast", "batch": 64, "hq": 64, "hkv": 8, "prefix": 4000,
         "tokens": 200},
        # The bounds of a long cache's pages.
        {"name": "bounds_32k", "op": "bounds", "layout": "default", "batch": 1, "hq": 32, "hkv": 8, "tokens": 32768},
        # And of a few pages that a chunk has filled, in the layout of make_turbo_caches.
        {"name": "bounds_1k", "op": "bounds", "layout": "fast", "batch": 1, "hq": 32, "hkv": 8, "tokens": 1024},
        # A step over a long chat, an eighth of its pages.
        {"name": "select_32k", "op": "select", "layout": "default", "batch": 1, "hq": 32, "hkv": 8, "tokens": 32805,
         "pages": 64, "first": 1, "last": 2},
        # The largest context, in the layout of make_turbo_caches.
        {"name": "select_131k", "op": "select", "layout": "fast", "batch": 1, "hq": 32, "hkv": 8, "tokens": 131072,
         "pages": 128, "first": 1, "last": 4},
        # A serving batch of long contexts.
        {"name": "select_batch", "op": "select", "layout": "default", "batch": 8, "hq": 32, "hkv": 8, "tokens": 24000,
         "pages": 48, "first": 2, "last": 2},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate"] * 4 + ["shared"] * 4 + ["select"] * 4 + ["bounds"])
    hq, hkv = rng.choice(HEADS)
    layout = rng.choice(["default"] * 3 + ["fast"] * 3 + ["deep2", "l1_8bit", "odd_split", "int8_angles4"])
    if op == "rotate":
        kind = rng.choice(["step", "prompt"])
        dtype = rng.choice(["float16", "bfloat16", "float32"])
        case = {"op": op, "kind": kind, "layout": layout, "dtype": dtype, "tables": rng.choice([dtype, "float32"]),
                "interleaved": rng.choice([False, False, True])}
        if kind == "step":
            new = rng.choice([1, 1, 1, 2, 5])
            tokens = _log_uniform(rng, 1, 2000) // PAGE * PAGE + rng.randint(1, PAGE - 1 - new)
            return dict(case, batch=_log_uniform(rng, 1, 48), hq=hq, hkv=hkv, tokens=tokens, new=new)
        batch = rng.choice([1, 1, 2, 3])
        return dict(case, batch=batch, hq=hq, hkv=hkv, tokens=0,
                    new=_log_uniform(rng, 2, max(40, 32773 * 12 // (hq // 4 + hkv + 4) // batch // (1 + (dtype == "float32")) // 2)))
    if op == "shared":
        prefix = _log_uniform(rng, 20, max(40, 32805 * 8 // max(hkv, 8)))
        # At most the multiplications and the pages of the largest listed cases.
        batch = max(1, min(_log_uniform(rng, 2, 64), 32 * 32 * 32805 // (prefix * hq)))
        return {"op": op, "layout": layout, "batch": batch, "hq": hq, "hkv": hkv, "prefix": prefix,
                "tokens": _log_uniform(rng, 1, max(2, 32 * 300 * 8 // (batch * hkv)))}
    batch = rng.choice([1, 1, 1, 2, 4, 8])
    most = 131072 * 8 // max(hkv, 8) // batch // (1 if layout in ("default", "fast") else 2)
    if op == "bounds":
        return {"op": op, "layout": layout, "batch": batch, "hq": hq, "hkv": hkv,
                "tokens": max(1, _log_uniform(rng, 64, max(128, most // 4)) // PAGE) * PAGE}
    tokens = _log_uniform(rng, 200, max(400, most))
    stored = tokens // PAGE
    pages = max(1, min(stored, _log_uniform(rng, 2, 256)))
    first = rng.randint(0, min(2, pages))
    return {"op": op, "layout": layout, "batch": batch, "hq": hq, "hkv": hkv, "tokens": tokens, "pages": pages,
            "first": first, "last": rng.randint(0, min(4, pages - first))}


# ---- inputs ---------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _row_bytes(layout):
    _, l1, deep, split = LAYOUTS[layout]
    return -(-(split // 2) * l1 // 8), -(-(PAIRS - split // 2) * deep // 8)


def _config(case):
    int8, l1, deep, split = LAYOUTS[case["layout"]]
    return {"num_q_heads": case["hq"], "num_kv_heads": case["hkv"], "use_int8_radii": int8, "k_angle_bits_level1": l1,
            "k_angle_bits_deep": deep, "split_dim": split}


def _pages(case, B, S, g):
    """Compressed pages of keys with per-channel scales and of normal values: radii of normal pairs, their log radii to
    8 bits of the page's largest where the layout has them, angles that drift from page to page as positions turn them,
    values to 8 bits of each group's largest."""
    int8, l1, deep, split = LAYOUTS[case["layout"]]
    H = case["hkv"]
    l1_row, deep_row = _row_bytes(case["layout"])
    channel = torch.exp((torch.rand((1, H, 1, 1, PAIRS), generator=g, device="cuda") * 2 - 1) * math.log(4.0))
    # Pages differ in size too: some hold what later queries look for.
    weight = torch.exp(0.5 * torch.randn((B, H, S, 1, 1), generator=g, device="cuda"))
    x = torch.randn((B, H, S, PAGE, DIM), generator=g, device="cuda")
    r = x.square().unflatten(-1, (PAIRS, 2)).sum(-1).sqrt() * channel * weight
    buffers = {}
    if int8:
        log = r.clamp(min=1e-3).log()
        scale = (log.abs().amax(dim=(-2, -1), keepdim=True) / 127).half()
        buffers["k.radii"] = (log / scale.float()).round().clamp(-127, 127).to(torch.int8)
        buffers["k.radii_scales"] = scale
    else:
        buffers["k.radii"] = r.half()
    for name, row in (("k.angle_l1", l1_row), ("k.angle_deep", deep_row)):
        if row:
            buffers[name] = torch.randint(0, 256, (B, H, S, PAGE, row), generator=g, device="cuda", dtype=torch.uint8)
    v = torch.randn((B, H, S, PAGE, 4, 32), generator=g, device="cuda")
    scales = (v.abs().amax(-1) / 127).half()
    buffers["v.codes"] = (v / scales.unsqueeze(-1).float()).round().clamp(-127, 127).to(torch.int8).flatten(-2).unsqueeze(3)
    buffers["v.scales"] = scales.unsqueeze(3)
    return buffers


def _cache(case, B, tokens, pages, tail_k, tail_v):
    """The cache that a serving program keeps, holding these pages and this tail."""
    from turbopolar_amd import TurboPolarFastCache, wire

    S, tail = tokens // PAGE, tokens % PAGE
    capacity = 4
    while capacity < S:
        capacity *= 2
    meta = {"format": "turbopolar-pages", "version": "1", "config": json.dumps(_config(case)), "batch": str(B),
            "kv_heads": str(case["hkv"]), "head_dim": str(DIM), "input_dtype": "torch.float16",
            "actual_seq_len": str(tokens), "pages": str(S), "tail_tokens": str(tail), "total_blocks": str(S),
            "bytes_written": "0", "bytes_read": "0", "compression_time_ns": "0"}
    for kind in "kv":
        meta.update({f"{kind}_capacity": str(capacity), f"{kind}_reallocs": "0", f"{kind}_growth_bytes": "0"})
    tensors = dict(pages)
    tensors.update({"tail.k": tail_k, "tail.v": tail_v})
    runtime = wire.load_state_dict(tensors, meta, "cuda:0")
    cache = TurboPolarFastCache(runtime.config)
    cache.runtime = runtime
    return cache


def _tables(case):
    """Cosines and sines of the new tokens' positions, as a model's rotary embedding hands them over: one angle a pair,
    both halves alike, or pairs side by side."""
    positions = torch.arange(case["tokens"], case["tokens"] + case["new"], dtype=torch.float64, device="cuda")
    turn = torch.pow(10000.0, -torch.arange(0, DIM, 2, dtype=torch.float64, device="cuda") / DIM)
    angle = positions[:, None] * turn
    angle = angle.repeat_interleave(2, -1) if case["interleaved"] else torch.cat((angle, angle), -1)
    dtype = getattr(torch, case["tables"])
    return angle.cos().to(dtype)[None], angle.sin().to(dtype)[None]


def _dense(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").half()


def prepare(case, seed):
    g = _generator(seed)
    B, hq, hkv = case["batch"], case["hq"], case["hkv"]
    state = {"case": case}
    if case["op"] == "rotate":
        dtype = getattr(torch, case["dtype"])
        channel = torch.exp((torch.rand((hkv, DIM), generator=g, device="cuda") * 2 - 1) * math.log(4.0))
        make = lambda h: torch.randn((B, case["new"], h, DIM), generator=g, device="cuda")  # noqa: E731
        # As the projections leave them: token by token.
        state.update(q=make(hq).to(dtype).transpose(1, 2), k=(make(hkv) * channel).to(dtype).transpose(1, 2),
                     v=make(hkv).to(dtype).transpose(1, 2))
        state["cos"], state["sin"] = _tables(case)
        if case["kind"] == "step":
            tail = case["tokens"] % PAGE
            pages = _pages(case, B, case["tokens"] // PAGE, g)
            for name in "kv":
                state["tail_" + name] = _dense(g, B, hkv, tail, DIM)
                # The tail as a buffer with room for a page, as a cache keeps it.
                state["room_" + name] = torch.zeros((B, hkv, PAGE, DIM), dtype=torch.float16, device="cuda")
                state["room_" + name][:, :, :tail] = state["tail_" + name]
            if own:
                state["cache"] = _cache(case, B, case["tokens"], pages, state["tail_k"], state["tail_v"])
        elif own:
            from turbopolar_amd import TurboPolarConfig

            state["config"] = TurboPolarConfig(**_config(case))
        return state
    if case["op"] == "shared":
        for name, rows, tokens in (("prefix", 1, case["prefix"]), ("own", B, case["tokens"])):
            state[name] = _pages(case, rows, tokens // PAGE, g)
            state[name + "_k"], state[name + "_v"] = (_dense(g, rows, hkv, tokens % PAGE, DIM) for _ in "kv")
        state["q"] = _dense(g, B, hq, 1, DIM)
        if own:
            from turbopolar_amd import SharedPrefixCache

            held = [_cache(case, rows, tokens, state[name], state[name + "_k"], state[name + "_v"])
                    for name, rows, tokens in (("prefix", 1, case["prefix"]), ("own", B, case["tokens"]))]
            state["cache"] = SharedPrefixCache(held[0], held[1])
        return state
    tokens, S = case["tokens"], case["tokens"] // PAGE
    state["pages"] = pages = _pages(case, B, S, g)
    state["tail_k"], state["tail_v"] = (_dense(g, B, hkv, tokens % PAGE, DIM) for _ in "kv")
    if case["op"] == "select":
        state["q"] = _dense(g, B, hq, DIM)
        state["bounds"] = _plain_bounds(state)
    if own:
        from turbopolar_amd import HipKernelBridge

        state["bridge"] = HipKernelBridge()
        state["cache"] = _cache(case, B, tokens, pages, state["tail_k"], state["tail_v"])
        state["block"], state["values"], *_ = state["cache"].runtime.get_fused_attention_inputs()
    return state


# ---- plain forms ----------------------------------------------------------------


def _scale():
    """1 / sqrt(128) as the kernels of this framework take it, an fp16 number."""
    return float(torch.tensor(1.0 / math.sqrt(DIM)).half())


def _codes(packed, bits, n):
    """The first n codes of a packed row, lowest bits of a byte first."""
    if bits == 8:
        return packed[..., :n].float()
    shifts = torch.arange(0, 8, bits, device=packed.device, dtype=torch.int32)
    codes = (packed.int().unsqueeze(-1) >> shifts) & (2 ** bits - 1)
    return codes.flatten(-2)[..., :n].float()


def _pair_keys(layout, codes, radii):
    """Keys from angle codes [..., 64] and radii, in 32 bits."""
    _, l1, deep, split = LAYOUTS[layout]
    levels = torch.full((PAIRS,), 2.0 ** deep - 1, device=codes.device)
    levels[:split // 2] = 2.0 ** l1 - 1
    angle = codes / levels * (2 * math.pi) - math.pi
    return torch.stack((radii * torch.cos(angle), radii * torch.sin(angle)), -1).flatten(-2)


def _plain_keys(layout, pages):
    """Keys [B, H, S, 64, 128] of compressed pages, in 32 bits."""
    int8, l1, deep, split = LAYOUTS[layout]
    codes = []
    if split:
        codes.append(_codes(pages["k.angle_l1"], l1, split // 2))
    if split < DIM:
        codes.append(_codes(pages["k.angle_deep"], deep, PAIRS - split // 2))
    radii = pages["k.radii"].float()
    if int8:
        radii = torch.exp(radii * pages["k.radii_scales"].float())
    return _pair_keys(layout, torch.cat(codes, -1), radii)


def _plain_values(pages):
    values = pages["v.codes"].float().unflatten(-1, (4, 32)) * pages["v.scales"].float().unsqueeze(-1)
    return values.flatten(-2).squeeze(3)


def _plain_bounds(state):
    keys = _plain_keys(state["case"]["layout"], state["pages"]).half()
    return torch.stack((keys.amin(3), keys.amax(3)), 3)


def _half64(x):
    """64-bit numbers rounded to fp16 once: to odd in 32 bits first, so that the second rounding decides."""
    f = x.float()
    over = f.double().abs() > x.abs()
    f = torch.where(over, torch.nextafter(f, torch.zeros_like(f)), f)
    bits = f.view(torch.int32)
    return torch.where(f.double() != x, bits | 1, bits).view(torch.float32).half()


def _rotate64(x, cos, sin, interleaved):
    """[B, H, T, 128] turned by [1, T, 128] tables, rounded to fp16 by way of 32 bits, as a cast does."""
    x, cos, sin = x.double(), cos.double().unsqueeze(1), sin.double().unsqueeze(1)
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        other = torch.stack((-b, a), -1).flatten(-2)
    else:
        other = torch.cat((-x[..., PAIRS:], x[..., :PAIRS]), -1)
    return (x * cos + other * sin).float().half()


def _encoded_keys(layout, k):
    """Keys [B, H, S, 64, 128] in fp16 through the page codec and back, in 32 bits: every step of the encoder's is
    rounded to fp16 (computed in 64 bits, rounded to 32 and to 16, which is one rounding for these)."""
    int8, l1, deep, split = LAYOUTS[layout]
    x, y = k[..., 0::2], k[..., 1::2]
    radii = ((x.float() * x.float()).half().float() + (y.float() * y.float()).half().float()).half()
    radii = radii.double().sqrt().float().half()
    shifted = (_half64(torch.atan2(y.double(), x.double())).float() + 3.140625).half()
    turn = (shifted.double() / 6.28125).float().half().float().clamp(0, 1)
    levels = torch.full((PAIRS,), 2.0 ** deep - 1, device=k.device)
    levels[:split // 2] = 2.0 ** l1 - 1
    codes = (turn * levels).round()
    if int8:
        floor = torch.tensor(1e-6, dtype=torch.float16, device=k.device)
        log = _half64(torch.maximum(radii, floor).double().log()).float()
        top = log.abs().amax((-2, -1), keepdim=True)
        top = torch.where(top == 0, torch.full_like(top, 1e-6), top)
        scale = (top.double() / 127).float().half().float()
        radii = torch.exp((log.double() / scale.double()).float().round().clamp(-128, 127) * scale)
    return _pair_keys(layout, codes, radii.float())


def _encoded_values(v):
    groups = v.unflatten(-1, (4, 32))
    scale = (groups.abs().amax(-1, keepdim=True).double() / 127).float().half()
    scale = torch.where(scale == 0, torch.full_like(scale, 1e-4), scale)
    codes = (groups.double() / scale.double()).float().half().float().round().clamp(-128, 127)
    return (codes * scale.float()).flatten(-2)


def _plain_rotate(state):
    case = state["case"]
    q = _rotate64(state["q"], state["cos"], state["sin"], case["interleaved"])
    k = _rotate64(state["k"], state["cos"], state["sin"], case["interleaved"])
    v = state["v"].half()
    if not (bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all())):
        raise ValueError("appended tokens must be finite")
    if case["kind"] == "step":
        tail = case["tokens"] % PAGE
        n = tail + case["new"]
        state["room_k"][:, :, tail:n], state["room_v"][:, :, tail:n] = k, v
        return {"q": q, "tail.k": state["room_k"][:, :, :n], "tail.v": state["room_v"][:, :, :n]}
    T = case["new"]
    pad = (0, 0, 0, -T % PAGE)
    k, v = (torch.nn.functional.pad(t, pad).unflatten(2, (-1, PAGE)) for t in (k, v))
    k, v = _encoded_keys(case["layout"], k).half(), _encoded_values(v).half()
    return {"q": q, "k": k.flatten(2, 3)[:, :, :T], "v": v.flatten(2, 3)[:, :, :T]}


def _softmax(scores):
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top)
    return weights / weights.sum(-1, keepdim=True)


def _plain_shared(state):
    case, q = state["case"], state["q"]
    B, hkv, g = case["batch"], case["hkv"], case["hq"] // case["hkv"]
    held = []
    for name in ("prefix", "own"):
        keys, values = _plain_keys(case["layout"], state[name]).flatten(2, 3), _plain_values(state[name]).flatten(2, 3)
        held.append((torch.cat((keys, state[name + "_k"].float()), 2), torch.cat((values, state[name + "_v"].float()), 2)))
    rows = q.float().squeeze(2).unflatten(1, (hkv, g))  # [B, hkv, g, 128]
    together = rows.transpose(0, 1).flatten(1, 2)  # [hkv, B * g, 128]: every row over the one prefix
    (pk, pv), (ok, ov) = held
    first = (together @ pk[0].transpose(-1, -2)).unflatten(1, (B, g)).transpose(0, 1)
    weights = _softmax(torch.cat((first, rows @ ok.transpose(-1, -2)), -1) * _scale())
    first, rest = weights.split((case["prefix"], case["tokens"]), -1)
    out = (first.transpose(0, 1).flatten(1, 2) @ pv[0]).unflatten(1, (B, g)).transpose(0, 1) + rest @ ov
    return out.flatten(1, 2).half()


def _plain_select(state):
    case, q = state["case"], state["q"]
    B, hkv, S, n = case["batch"], case["hkv"], case["tokens"] // PAGE, case["pages"]
    rows = q.unflatten(1, (hkv, -1)).double()  # [B, hkv, g, 128]
    low, high = state["bounds"].double().unsqueeze(2).unbind(4)  # [B, hkv, 1, S, 128]
    best = None
    for h in range(rows.shape[2]):
        x = rows[:, :, h:h + 1, None]
        s = torch.maximum(x * low, x * high).sum(-1).squeeze(2)
        best = s if best is None else torch.maximum(best, s)
    best[:, :, :case["first"]] = math.inf
    best[:, :, S - case["last"]:] = math.inf
    order = torch.sort(best, dim=-1, descending=True, stable=True).indices[..., :n]
    chosen = order.sort(-1).values  # [B, hkv, n]
    at = (torch.arange(B, device=q.device)[:, None, None], torch.arange(hkv, device=q.device)[:, None], chosen)
    pages = {name: t[at] for name, t in state["pages"].items()}
    keys = torch.cat((_plain_keys(case["layout"], pages).flatten(2, 3), state["tail_k"].float()), 2)
    values = torch.cat((_plain_values(pages).flatten(2, 3), state["tail_v"].float()), 2)
    weights = _softmax(rows.float() @ keys.transpose(-1, -2) * _scale())
    return {"selected": chosen.int(), "out": (weights @ values).flatten(1, 2).half()}


# ---- one pass ----------------------------------------------------------------------


def _run_own(state):
    case = state["case"]
    if case["op"] == "rotate":
        inputs = (state["q"], state["k"], state["v"], state["cos"], state["sin"], case["interleaved"])
        if case["kind"] == "prompt":
            from turbopolar_amd import TurboPolarFastCache

            q, k, v = TurboPolarFastCache(state["config"]).update_rotated(*inputs)
            return {"q": q, "k": k, "v": v}
        cache = state["cache"]
        q = cache.append_rotated(*inputs)
        _, _, tail_k, tail_v, _, _ = cache.runtime.get_fused_attention_inputs()
        cache.truncate(case["tokens"])
        return {"q": q, "tail.k": tail_k, "tail.v": tail_v}
    if case["op"] == "shared":
        return state["cache"].attention(state["q"], state["cache"].config.attention_scale)
    if case["op"] == "bounds":
        return state["bridge"].execute_page_bounds(state["block"])[0]
    out, trace = state["bridge"].execute_selected_attention_quant_v_dense_tail(
        state["q"], state["block"], state["values"], state["bounds"], state["tail_k"], state["tail_v"],
        state["cache"].config, pages=case["pages"], first=case["first"], last=case["last"])
    return {"selected": trace["selected"], "out": out}


def run(state):
    if own:
        return _run_own(state)
    return {"rotate": _plain_rotate, "shared": _plain_shared, "bounds": _plain_bounds, "select": _plain_select}[
        state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------


def _page_bytes(layout, values=True):
    l1_row, deep_row = _row_bytes(layout)
    int8 = LAYOUTS[layout][0]
    return PAGE * (PAIRS * (1 if int8 else 2) + l1_row + deep_row + (DIM + 8 if values else 0)) + (2 if int8 else 0)


def work(case):
    B, hq, hkv = case["batch"], case["hq"], case["hkv"]
    page, token = _page_bytes(case["layout"]), 4 * DIM  # of a dense token: its key and value
    if case["op"] == "rotate":
        T = case["new"]
        size, table = (4 if case[n] == "float32" else 2 for n in ("dtype", "tables"))
        moved = B * T * DIM * (hq * (size + 2) + 2 * hkv * size) + 2 * T * DIM * table
        if case["kind"] == "step":
            return {"bytes": moved + B * T * hkv * token, "flops": 3 * B * T * DIM * (hq + hkv)}
        return {"bytes": moved + B * hkv * (T // PAGE * page + T % PAGE * token) + B * hkv * T * token,
                "flops": 3 * B * T * DIM * (hq + hkv)}
    if case["op"] == "shared":
        held = [n // PAGE * page + n % PAGE * token for n in (case["prefix"], case["tokens"])]
        return {"bytes": hkv * (held[0] + B * held[1]) + B * hq * 4 * DIM,
                "flops": 4 * DIM * B * hq * (case["prefix"] + case["tokens"])}
    S = case["tokens"] // PAGE
    if case["op"] == "bounds":
        return {"bytes": B * hkv * S * (_page_bytes(case["layout"], False) + 4 * DIM), "flops": 4 * B * hkv * S * PAGE * DIM}
    n, tail = case["pages"], case["tokens"] % PAGE
    return {"bytes": B * hkv * (S * 4 * DIM + n * (page + 4) + tail * token) + B * hq * 4 * DIM,
            "flops": B * hq * 4 * DIM * (S + n * PAGE + tail)}


# ---- the same in 64 bits, from the definitions ------------------------------------------


def _decode64(layout, pages, b, h):
    """Keys and values of one (batch, head) in 64 bits, [pages * 64, 128] each."""
    int8, l1, deep, split = LAYOUTS[layout]
    at = {name: t[b, h] for name, t in pages.items()}
    angle = torch.empty(at["k.radii"].shape, dtype=torch.float64, device="cuda")
    for pair in range(PAIRS):
        row, bits, i = ("k.angle_l1", l1, pair) if pair < split // 2 else ("k.angle_deep", deep, pair - split // 2)
        byte = at[row][..., i * bits // 8].long()
        angle[..., pair] = ((byte >> (i * bits % 8)) % 2 ** bits).double() / (2 ** bits - 1) * 2 * math.pi - math.pi
    r = at["k.radii"].double()
    if int8:
        r = (r * at["k.radii_scales"].double()).exp()
    keys = torch.empty(*r.shape[:-1], DIM, dtype=torch.float64, device="cuda")
    keys[..., 0::2], keys[..., 1::2] = r * angle.cos(), r * angle.sin()
    values = at["v.codes"].double() * at["v.scales"].double().repeat_interleave(32, -1)
    return keys.reshape(-1, DIM), values.reshape(-1, DIM)


def _attend64(q, k, v):
    s = q @ k.T * float(torch.tensor(DIM ** -0.5, dtype=torch.float64).to(torch.float16))
    return torch.softmax(s, -1) @ v


def _exact_shared(state):
    case = state["case"]
    g = case["hq"] // case["hkv"]
    out = torch.empty((case["batch"], case["hq"], DIM), dtype=torch.float64, device="cuda")
    for h in range(case["hkv"]):
        pk, pv = _decode64(case["layout"], state["prefix"], 0, h)
        for b in range(case["batch"]):
            k, v = _decode64(case["layout"], state["own"], b, h)
            k = torch.cat((pk, state["prefix_k"][0, h].double(), k, state["own_k"][b, h].double()))
            v = torch.cat((pv, state["prefix_v"][0, h].double(), v, state["own_v"][b, h].double()))
            heads = slice(h * g, (h + 1) * g)
            out[b, heads] = _attend64(state["q"][b, heads, 0].double(), k, v)
    return out


def _exact_select(state):
    case = state["case"]
    hkv, S, n = case["hkv"], case["tokens"] // PAGE, case["pages"]
    g = case["hq"] // hkv
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    chosen = torch.empty((case["batch"], hkv, n), dtype=torch.int32)
    for b in range(case["batch"]):
        for h in range(hkv):
            heads = slice(h * g, (h + 1) * g)
            q, (low, high) = state["q"][b, heads].double(), state["bounds"][b, h].double().unbind(1)
            scores = (q.clamp(min=0) @ high.T + q.clamp(max=0) @ low.T).amax(0).tolist()
            forced = [i < case["first"] or i >= S - case["last"] for i in range(S)]
            pick = sorted(sorted(range(S), key=lambda i: (not forced[i], -scores[i], i))[:n])
            chosen[b, h] = torch.tensor(pick, dtype=torch.int32)
            pages = {name: t[b:b + 1, h:h + 1, pick] for name, t in state["pages"].items()}
            k, v = _decode64(case["layout"], pages, 0, 0)
            out[b, heads] = _attend64(q, torch.cat((k, state["tail_k"][b, h].double())),
                                      torch.cat((v, state["tail_v"][b, h].double())))
    return {"selected": chosen.cuda(), "out": out}


def _exact_rotate(state):
    """The rotation in 64 bits; of a prompt's history, whose codes are chosen from its rotated keys in fp16, what the
    codes stand for."""
    case = state["case"]
    sides = {}
    for name in "qk":
        x, c, s = state[name].double(), state["cos"][0].double(), state["sin"][0].double()
        y = torch.empty_like(x)
        a, b = (slice(0, None, 2), slice(1, None, 2)) if case["interleaved"] else (slice(0, PAIRS), slice(PAIRS, DIM))
        y[..., a] = x[..., a] * c[:, a] - x[..., b] * s[:, a]
        y[..., b] = x[..., b] * c[:, b] + x[..., a] * s[:, b]
        sides[name] = y
    v = state["v"].double()
    if case["kind"] == "step":
        return {"q": sides["q"], "tail.k": torch.cat((state["tail_k"].double(), sides["k"]), 2),
                "tail.v": torch.cat((state["tail_v"].double(), v), 2)}
    int8, l1, deep, split = LAYOUTS[case["layout"]]
    B, H, T, _ = v.shape
    if B * H * T > 400000:
        return {"q": sides["q"], "k": None, "v": None}
    half = lambda t: t.float().half().cpu().numpy()  # noqa: E731
    k16, v16 = (np.zeros((B, H, -(-T // PAGE), PAGE, DIM), np.float16) for _ in "kv")
    k16.reshape(B, H, -1, DIM)[:, :, :T], v16.reshape(B, H, -1, DIM)[:, :, :T] = half(sides["k"]), half(v)
    x, y = k16[..., 0::2], k16[..., 1::2]
    with np.errstate(over="ignore"):
        r = np.sqrt(x * x + y * y)
    turn = np.arctan2(y.astype(np.float64), x.astype(np.float64)).astype(np.float16)
    turn = np.clip((turn + np.float16(np.pi)) / np.float16(2 * np.pi), np.float16(0), np.float16(1)).astype(np.float32)
    top = np.where(np.arange(PAIRS) < split // 2, 2 ** l1 - 1, 2 ** deep - 1)
    angle = np.rint(turn * top.astype(np.float32)).astype(np.float64) / top * 2 * np.pi - np.pi
    size = r.astype(np.float64)
    if int8:
        log = np.log(np.maximum(r, np.float16(1e-6)).astype(np.float64)).astype(np.float16).astype(np.float32)
        step = np.abs(log).max((-2, -1), keepdims=True)
        step = (np.where(step == 0, np.float32(1e-6), step) / np.float32(127)).astype(np.float16).astype(np.float32)
        size = np.exp(np.clip(np.rint(log / step), -128, 127).astype(np.float64) * step)
    keys = np.stack((size * np.cos(angle), size * np.sin(angle)), -1)
    groups = v16.reshape(*v16.shape[:-1], 4, 32)
    step = np.abs(groups).max(-1, keepdims=True) / np.float16(127)
    step = np.where(step == 0, np.float16(1e-4), step)
    values = np.clip(np.rint(groups / step), -128, 127).astype(np.float64) * step
    back = lambda t: torch.from_numpy(np.ascontiguousarray(t.reshape(B, H, -1, DIM)[:, :, :T])).cuda()  # noqa: E731
    return {"q": sides["q"], "k": back(keys), "v": back(values)}


def exact(case, seed):
    global own
    kept, own = own, False  # the inputs alone
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "shared":
        return _exact_shared(state)
    if case["op"] == "select":
        return _exact_select(state)
    if case["op"] == "rotate":
        return _exact_rotate(state)
    out = torch.empty((case["batch"], case["hkv"], case["tokens"] // PAGE, 2, DIM), dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        for h in range(case["hkv"]):
            keys = _decode64(case["layout"], state["pages"], b, h)[0].reshape(-1, PAGE, DIM)
            out[b, h, :, 0], out[b, h, :, 1] = keys.amin(1), keys.amax(1)
    return out
