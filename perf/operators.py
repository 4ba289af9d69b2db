"""Operators of a serving loop around a compressed cache, as timed cases with their plain forms.

``op`` names what one pass does:

* ``prompt``  attention of a whole prompt (or of a chunk after a dense history), causal or not, grouped query
  heads, sequences of one length or packed ones of different lengths;
* ``tree``    attention of a tree of drafted tokens over a compressed cache: every node sees the stored pages, the
  dense tail and its ancestors among the drafted tokens;
* ``fork``    a cache copied: whole, chosen batch rows of it, chosen pages, or the first tokens;
* ``accept``  the accepted path of a draft compacted into the cache, and the cache taken back to its length.

With ``own`` false ``run`` computes them in elementary torch operations in 32 bits; with ``own`` true it makes the
calls of this repository's package.
"""

import json
import math
import random

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
        # A chat turn's prompt: a couple of hundred tokens, where latency counts.
        {"name": "prompt_200", "op": "prompt", "dtype": "float16", "batch": 1, "hq": 32, "hkv": 8, "tq": 200, "tk": 200,
         "causal": True, "sequences": 0, "mix": 0},
        # An ordinary prompt of the benchmark's shape.
        {"name": "prompt_4k", "op": "prompt", "dtype": "float16", "batch": 1, "hq": 32, "hkv": 8, "tq": 4096,
         "tk": 4096, "causal": True, "sequences": 0, "mix": 0},
        # A long document at once, in bfloat16.
        {"name": "prompt_16k", "op": "prompt", "dtype": "bfloat16", "batch": 1, "hq": 32, "hkv": 8, "tq": 16384,
         "tk": 16384, "causal": True, "sequences": 0, "mix": 0},
        # The prompts of several users packed into one row of tokens, seven query heads a group, spare rows behind.
        {"name": "prompt_packed", "op": "prompt", "dtype": "bfloat16", "batch": 1, "hq": 28, "hkv": 4, "tq": 8100,
         "tk": 8100, "causal": True, "sequences": 23, "mix": 5},
        # The next chunk of a prompt, after a history that was decompressed.
        {"name": "prompt_chunk", "op": "prompt", "dtype": "float16", "batch": 1, "hq": 32, "hkv": 8, "tq": 500,
         "tk": 8600, "causal": True, "sequences": 0, "mix": 0},
        # A small draft early in a chat, where latency counts.
        {"name": "tree_1k", "op": "tree", "layout": "default", "batch": 1, "hq": 32, "hkv": 8, "tokens": 1000,
         "nodes": 8, "shape": "tree"},
        # A draft of 32 nodes over the benchmark's context, between two page flushes.
        {"name": "tree_32k", "op": "tree", "layout": "default", "batch": 1, "hq": 32, "hkv": 8, "tokens": 32805,
         "nodes": 32, "shape": "tree"},
        # A serving batch, eight query heads a group, in the layout of make_turbo_caches.
        {"name": "tree_batch", "op": "tree", "layout": "fast", "batch": 8, "hq": 64, "hkv": 8, "tokens": 4000,
         "nodes": 16, "shape": "tree"},
        # A short drafted chain over the largest context.
        {"name": "tree_131k", "op": "tree", "layout": "fast", "batch": 1, "hq": 32, "hkv": 8, "tokens": 131072,
         "nodes": 5, "shape": "chain"},
        # A branch of a long conversation: the whole cache copied.
        {"name": "fork_32k", "op": "fork", "layout": "default", "batch": 1, "hq": 32, "hkv": 8, "tokens": 32805,
         "rows": 0, "keep": 0, "pages": 0},
        # A batch of hypotheses re-ordered and taken back to a common prefix that ends inside a page.
        {"name": "fork_rows", "op": "fork", "layout": "fast", "batch": 8, "hq": 32, "hkv": 8, "tokens": 4000,
         "rows": 8, "keep": 3777, "pages": 0},
        # The end of a drafted step: five accepted tokens into a 300-token cache.
        {"name": "accept_5", "op": "accept", "layout": "fast", "batch": 1, "hq": 32, "hkv": 8, "tokens": 300,
         "nodes": 16, "shape": "tree", "path": 5},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt"] * 5 + ["tree"] * 5 + ["fork"] * 2 + ["accept"])
    hq, hkv = rng.choice(HEADS)
    if op == "prompt":
        # At most the multiplications of the largest listed case.
        tk = _log_uniform(rng, 1, min(16384, int(16384 * math.sqrt(32 / hq))))
        batch = rng.choice([1, 1, 1, 2, 3]) if tk < 6000 else 1
        kind = rng.choice(["whole", "whole", "packed", "chunk", "full"])
        tq = max(1, tk // rng.randint(2, 40)) if kind == "chunk" else tk
        packed = kind == "packed" and tk >= 8
        return {"op": op, "dtype": rng.choice(["float16", "bfloat16"]), "batch": 1 if packed else batch, "hq": hq,
                "hkv": hkv, "tq": tq, "tk": tk, "causal": kind != "full",
                "sequences": rng.randint(2, min(32, tk // 4)) if packed else 0,
                "mix": rng.randint(1, 1000) if packed else 0}
    layout = rng.choice(["default"] * 3 + ["fast"] * 3 + ["deep2", "l1_8bit", "odd_split", "int8_angles4"])
    if op == "tree":
        batch = rng.choice([1, 1, 1, 2, 4, 8])
        tokens = _log_uniform(rng, 20, max(40, 131072 * 8 // max(hkv, 8) // batch // (1 if layout in ("default", "fast") else 4)))
        most = max(1, min(64, 4 * 32805 * 32 // (tokens * batch * hq // hkv)))
        return {"op": op, "layout": layout, "batch": batch, "hq": hq, "hkv": hkv, "tokens": tokens,
                "nodes": _log_uniform(rng, 1, most), "shape": rng.choice(["tree", "chain"])}
    batch = rng.choice([1, 2, 4, 8])
    tokens = _log_uniform(rng, 65, max(130, 32805 * 8 // max(hkv, 8) // batch))
    if op == "fork":
        kind = rng.choice(["whole", "rows", "prefix", "pages"])
        return {"op": op, "layout": layout, "batch": batch, "hq": hq, "hkv": hkv, "tokens": tokens,
                "rows": rng.randint(1, 8) if kind == "rows" else 0,
                "keep": rng.randint(1, tokens) if kind == "prefix" else 0,
                "pages": rng.randint(1, tokens // PAGE) if kind == "pages" else 0}
    nodes = rng.randint(2, 64)
    path = rng.randint(1, min(8, nodes))
    # The path ends before a page is full, so that the cache can be taken back to its length exactly.
    tokens = tokens // PAGE * PAGE + rng.randint(1, PAGE - 1 - path)
    return {"op": op, "layout": layout, "batch": batch, "hq": hq, "hkv": hkv, "tokens": tokens, "nodes": nodes,
            "shape": rng.choice(["tree", "chain"]), "path": path}


# ---- inputs ---------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _starts(case):
    """First tokens of packed sequences, and the end of the last: lengths over the whole range, one of a single token,
    and some rows behind the last sequence."""
    rng = random.Random(case["mix"])
    n = case["sequences"]
    rest = case["tk"] // 90
    weights = [math.exp(rng.uniform(0, 4)) for _ in range(n)]
    room = case["tk"] - rest - n
    lengths = [1 + int(room * w / sum(weights)) for w in weights]
    lengths[rng.randrange(n)] = 1
    starts = [0]
    for x in lengths:
        starts.append(starts[-1] + x)
    return starts


def _parents(case, seed):
    """Parent of each drafted token (-1: the cache's last token)."""
    n = case["nodes"]
    if case["shape"] == "chain":
        return list(range(-1, n - 1))
    rng = random.Random(seed)
    return [-1] + [rng.randrange(max(-1, i - 6), i) for i in range(1, n)]


def _path(case, parents, seed):
    """An accepted path of the tree, and further nodes in order where the tree is not deep enough."""
    children, node, path = {}, -1, []
    for i, p in enumerate(parents):
        children.setdefault(p, []).append(i)
    rng = random.Random(seed + 1)
    while len(path) < case["path"] and children.get(node):
        node = rng.choice(children[node])
        path.append(node)
    path += [i for i in range(len(parents)) if i not in path][: case["path"] - len(path)]
    return path


def _row_bytes(layout):
    _, l1, deep, split = LAYOUTS[layout]
    return -(-(split // 2) * l1 // 8), -(-(PAIRS - split // 2) * deep // 8)


def _pages(case, g):
    """Compressed pages of keys with per-channel scales and of normal values: radii of normal pairs, their log radii
    to 8 bits of the page's largest where the layout has them, uniform angles, values to 8 bits of each group's largest."""
    int8, l1, deep, split = LAYOUTS[case["layout"]]
    B, H, S = case["batch"], case["hkv"], case["tokens"] // PAGE
    l1_row, deep_row = _row_bytes(case["layout"])
    channel = torch.exp((torch.rand((1, H, 1, 1, PAIRS), generator=g, device="cuda") * 2 - 1) * math.log(4.0))
    x = torch.randn((B, H, S, PAGE, DIM), generator=g, device="cuda")
    r = x.square().unflatten(-1, (PAIRS, 2)).sum(-1).sqrt() * channel
    buffers = {}
    if int8:
        log = r.clamp(min=1e-3).log()
        scale = (log.abs().amax(dim=(-2, -1), keepdim=True) / 127).half()
        buffers["k.radii"] = (log / scale.float()).round().clamp(-127, 127).to(torch.int8)
        buffers["k.radii_scales"] = scale
    else:
        buffers["k.radii"] = r.half()
    if l1_row:
        buffers["k.angle_l1"] = torch.randint(0, 256, (B, H, S, PAGE, l1_row), generator=g, device="cuda", dtype=torch.uint8)
    if deep_row:
        buffers["k.angle_deep"] = torch.randint(0, 256, (B, H, S, PAGE, deep_row), generator=g, device="cuda",
                                                dtype=torch.uint8)
    v = torch.randn((B, H, S, PAGE, 4, 32), generator=g, device="cuda")
    scales = (v.abs().amax(-1) / 127).half()
    buffers["v.codes"] = (v / scales.unsqueeze(-1).float()).round().clamp(-127, 127).to(torch.int8).flatten(-2).unsqueeze(3)
    buffers["v.scales"] = scales.unsqueeze(3)
    return buffers


def _cache(case, pages, tail_k, tail_v):
    """The cache that a serving program keeps, holding these pages and this tail."""
    from turbopolar_amd import TurboPolarFastCache, wire

    int8, l1, deep, split = LAYOUTS[case["layout"]]
    S, tail = case["tokens"] // PAGE, case["tokens"] % PAGE
    capacity = 4
    while capacity < S:
        capacity *= 2
    config = {"num_q_heads": case["hq"], "num_kv_heads": case["hkv"], "use_int8_radii": int8, "k_angle_bits_level1": l1,
              "k_angle_bits_deep": deep, "split_dim": split}
    meta = {"format": "turbopolar-pages", "version": "1", "config": json.dumps(config), "batch": str(case["batch"]),
            "kv_heads": str(case["hkv"]), "head_dim": str(DIM), "input_dtype": "torch.float16",
            "actual_seq_len": str(case["tokens"]), "pages": str(S), "tail_tokens": str(tail), "total_blocks": str(S),
            "bytes_written": "0", "bytes_read": "0", "compression_time_ns": "0"}
    for kind in "kv":
        meta.update({f"{kind}_capacity": str(capacity), f"{kind}_reallocs": "0", f"{kind}_growth_bytes": "0"})
    tensors = dict(pages)
    tensors.update({"tail.k": tail_k, "tail.v": tail_v})
    runtime = wire.load_state_dict(tensors, meta, "cuda:0")
    cache = TurboPolarFastCache(runtime.config)
    cache.runtime = runtime
    return cache


def prepare(case, seed):
    g = _generator(seed)
    B, hq, hkv = case["batch"], case["hq"], case["hkv"]
    if case["op"] == "prompt":
        dtype = getattr(torch, case["dtype"])
        channel = torch.exp((torch.rand((1, hkv, 1, DIM), generator=g, device="cuda") * 2 - 1) * math.log(2.0))
        state = {"case": case,
                 "q": torch.randn((B, hq, case["tq"], DIM), generator=g, device="cuda").to(dtype),
                 "k": (torch.randn((B, hkv, case["tk"], DIM), generator=g, device="cuda") * channel).to(dtype),
                 "v": torch.randn((B, hkv, case["tk"], DIM), generator=g, device="cuda").to(dtype)}
        if case["sequences"]:
            state["starts"] = torch.tensor(_starts(case), dtype=torch.int32, device="cuda")
        if own:
            from turbopolar_amd import HipKernelBridge, TurboPolarConfig

            state["bridge"], state["config"] = HipKernelBridge(), TurboPolarConfig(num_q_heads=hq, num_kv_heads=hkv)
        return state
    pages = _pages(case, g)
    dense = lambda heads, tokens: torch.randn((B, heads, tokens, DIM), generator=g, device="cuda").half()  # noqa: E731
    tail = case["tokens"] % PAGE
    state = {"case": case, "pages": pages, "tail_k": dense(hkv, tail), "tail_v": dense(hkv, tail)}
    if case["op"] in ("tree", "accept"):
        n = case["nodes"]
        parents = _parents(case, seed)
        state.update(k=dense(hkv, n), v=dense(hkv, n))
        if case["op"] == "tree":
            state["q"] = dense(hq, n)
            mask = torch.zeros((n, n), dtype=torch.bool)
            for i, p in enumerate(parents):
                if p >= 0:
                    mask[i] = mask[p]
                mask[i, i] = True
            state["mask"] = mask.cuda()
        else:
            state["path"] = _path(case, parents, seed)
            # The tail as a buffer with room for a page, as a cache keeps it.
            for name in ("tail_k", "tail_v"):
                state["room_" + name] = torch.zeros((B, hkv, PAGE, DIM), dtype=torch.float16, device="cuda")
                state["room_" + name][:, :, :tail] = state[name]
    elif case["rows"]:
        state["rows"] = [random.Random(seed).randrange(B) for _ in range(case["rows"])]
    elif case["pages"]:
        state["keep_pages"] = sorted(random.Random(seed).sample(range(case["tokens"] // PAGE), case["pages"]))
    if own:
        state["cache"] = _cache(case, pages, state["tail_k"], state["tail_v"])
        if case["op"] == "tree":
            from turbopolar_amd import DraftTree

            state["tree"] = DraftTree(parents, device="cuda:0")
    return state


# ---- plain forms ----------------------------------------------------------------


def _softmax_rows(scores, seen):
    """Softmax along the last axis over what is seen; a row that sees nothing is zero."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    return weights / torch.where(total == 0, torch.ones_like(total), total)


def _scale():
    """1 / sqrt(128) as the kernels of this framework take it, an fp16 number."""
    return float(torch.tensor(1.0 / math.sqrt(DIM)).half())


def _plain_prompt(state):
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    B, hq, tq, _ = q.shape
    hkv, tk = k.shape[1], k.shape[2]
    rows = torch.arange(tq, device=q.device)
    begin, end = torch.zeros_like(rows), torch.full_like(rows, tk)
    if case["sequences"]:
        starts = state["starts"].long()
        at = torch.bucketize(rows, starts[1:], right=True)
        live = at < case["sequences"]
        at = at.clamp(max=case["sequences"] - 1)
        begin, end = starts[at], torch.where(live, rows + 1, starts[at])
    elif case["causal"]:
        end = rows + (tk - tq + 1)
    keys, values = k.float().unsqueeze(2), v.float().unsqueeze(2)
    columns = torch.arange(tk, device=q.device)
    out = torch.empty_like(q)
    step = max(1, (1 << 29) // (B * hq * tk))  # at most 2 GiB of scores at a time
    for t in range(0, tq, step):
        part = q[:, :, t:t + step].float().unflatten(1, (hkv, hq // hkv))
        seen = (columns >= begin[t:t + step, None]) & (columns < end[t:t + step, None])
        weights = _softmax_rows(part @ keys.transpose(-1, -2) * _scale(), seen)
        out[:, :, t:t + step] = (weights @ values).flatten(1, 2).to(q.dtype)
    return out


def _codes(packed, bits, n):
    """The first n codes of a packed row, lowest bits of a byte first."""
    if bits == 8:
        return packed[..., :n].float()
    shifts = torch.arange(0, 8, bits, device=packed.device, dtype=torch.int32)
    codes = (packed.int().unsqueeze(-1) >> shifts) & (2 ** bits - 1)
    return codes.flatten(-2)[..., :n].float()


def _plain_decode(layout, pages):
    """Keys and values [B, H, S * 64, 128] of compressed pages, in 32 bits."""
    int8, l1, deep, split = LAYOUTS[layout]
    turns = []
    if split:
        turns.append(_codes(pages["k.angle_l1"], l1, split // 2) / (2 ** l1 - 1))
    if split < DIM:
        turns.append(_codes(pages["k.angle_deep"], deep, PAIRS - split // 2) / (2 ** deep - 1))
    angle = torch.cat(turns, -1) * (2 * math.pi) - math.pi
    radii = pages["k.radii"].float()
    if int8:
        radii = torch.exp(radii * pages["k.radii_scales"].float())
    keys = torch.stack((radii * torch.cos(angle), radii * torch.sin(angle)), -1).flatten(-2)
    values = pages["v.codes"].float().unflatten(-1, (4, 32)) * pages["v.scales"].float().unsqueeze(-1)
    return keys.flatten(2, 3), values.flatten(-2).squeeze(3).flatten(2, 3)


def _plain_tree(state):
    case, q = state["case"], state["q"]
    keys, values = _plain_decode(case["layout"], state["pages"])
    keys = torch.cat((keys, state["tail_k"].float(), state["k"].float()), 2).unsqueeze(2)
    values = torch.cat((values, state["tail_v"].float(), state["v"].float()), 2).unsqueeze(2)
    n = case["nodes"]
    seen = torch.cat((torch.ones((n, case["tokens"]), dtype=torch.bool, device=q.device), state["mask"]), 1)
    scores = q.float().unflatten(1, (case["hkv"], -1)) @ keys.transpose(-1, -2) * _scale()
    return (_softmax_rows(scores, seen) @ values).flatten(1, 2).half()


def _plain_fork(state):
    case, pages, tail_k, tail_v = state["case"], state["pages"], state["tail_k"], state["tail_v"]
    S, tail = case["tokens"] // PAGE, case["tokens"] % PAGE
    rows = torch.tensor(state["rows"], device="cuda") if case["rows"] else torch.arange(case["batch"], device="cuda")
    if case["keep"]:
        n, left = case["keep"] // PAGE, case["keep"] % PAGE
        chosen = torch.arange(n, device="cuda")
        if n < S and left:
            keys, values = _plain_decode(case["layout"], {name: t[:, :, n:n + 1] for name, t in pages.items()})
            tail_k, tail_v = keys[:, :, :left].half(), values[:, :, :left].half()
        else:
            tail_k, tail_v = tail_k[:, :, :left], tail_v[:, :, :left]
    elif case["pages"]:
        chosen = torch.tensor(state["keep_pages"], device="cuda")
    else:
        chosen = torch.arange(S, device="cuda")
    out = {name: t[rows[:, None], :, chosen[None, :]].transpose(1, 2).contiguous() for name, t in pages.items()}
    out["tail.k"], out["tail.v"] = tail_k[rows].contiguous(), tail_v[rows].contiguous()
    return out


def _plain_accept(state):
    case, tail = state["case"], state["case"]["tokens"] % PAGE
    path = torch.tensor(state["path"], device="cuda")
    k, v = state["k"][:, :, path], state["v"][:, :, path]
    if not (bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all())):
        raise ValueError("drafted tokens must be finite")
    n = tail + case["path"]
    state["room_tail_k"][:, :, tail:n], state["room_tail_v"][:, :, tail:n] = k, v
    return {"tail.k": state["room_tail_k"][:, :, :n], "tail.v": state["room_tail_v"][:, :, :n]}


# ---- one pass ----------------------------------------------------------------------


def _run_own(state):
    case = state["case"]
    if case["op"] == "prompt":
        starts = state.get("starts")
        out, _ = state["bridge"].execute_prompt_attention(state["q"], state["k"], state["v"], state["config"],
                                                          causal=case["causal"], q_starts=starts, k_starts=starts)
        return out
    cache = state["cache"]
    if case["op"] == "tree":
        return cache.tree_attention(state["q"], state["k"], state["v"], state["tree"], cache.config.attention_scale)
    if case["op"] == "fork":
        other = cache.fork(tokens=case["keep"] or None, rows=state.get("rows"), pages=state.get("keep_pages"))
        key, value, tail_k, tail_v, _, _ = other.runtime.get_fused_attention_inputs()
        none = state["tail_k"][:, :, :0]
        out = {"tail.k": none if tail_k is None else tail_k, "tail.v": none if tail_v is None else tail_v}
        for name in state["pages"]:
            t = state["pages"][name][:, :, :0] if key is None else {
                "k.radii": key.radii, "k.radii_scales": key.radii_scales, "k.angle_l1": key.angle_codes_l1,
                "k.angle_deep": key.angle_codes_deep, "v.codes": value.codes.unsqueeze(3),
                "v.scales": value.scales.unsqueeze(3)}[name]
            out[name] = t
        return out
    cache.accept(state["k"], state["v"], state["path"])
    _, _, tail_k, tail_v, _, _ = cache.runtime.get_fused_attention_inputs()
    cache.truncate(case["tokens"])
    return {"tail.k": tail_k, "tail.v": tail_v}


def run(state):
    if own:
        return _run_own(state)
    return {"prompt": _plain_prompt, "tree": _plain_tree, "fork": _plain_fork, "accept": _plain_accept}[
        state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------


def _page_bytes(layout):
    l1_row, deep_row = _row_bytes(layout)
    int8 = LAYOUTS[layout][0]
    return PAGE * (PAIRS * (1 if int8 else 2) + l1_row + deep_row + DIM + 8) + (2 if int8 else 0)


def work(case):
    B, hq, hkv = case["batch"], case["hq"], case["hkv"]
    if case["op"] == "prompt":
        tq, tk = case["tq"], case["tk"]
        if case["sequences"]:
            starts = _starts(case)
            pairs = sum(n * (n + 1) // 2 for n in (b - a for a, b in zip(starts, starts[1:])))
        else:
            pairs = tq * tk - (tq * (tq - 1) // 2 if case["causal"] else 0)
        return {"bytes": B * 2 * DIM * (2 * hq * tq + 2 * hkv * tk), "flops": 4 * DIM * B * hq * pairs}
    S, tail = case["tokens"] // PAGE, case["tokens"] % PAGE
    page = _page_bytes(case["layout"])
    token = 4 * DIM  # a dense token's key and value
    if case["op"] == "tree":
        n = case["nodes"]
        return {"bytes": B * hkv * (S * page + (tail + n) * token) + B * hq * n * 4 * DIM,
                "flops": 4 * DIM * B * hq * n * (case["tokens"] + n)}
    if case["op"] == "fork":
        rows = case["rows"] or B
        kept, left, decoded = S, tail, 0
        if case["keep"]:
            kept, left = case["keep"] // PAGE, case["keep"] % PAGE
            decoded = page if kept < S and left else 0
        elif case["pages"]:
            kept = case["pages"]
        return {"bytes": 2 * rows * hkv * (kept * page + left * token) + rows * hkv * decoded,
                "flops": rows * hkv * (8 * DIM * left if decoded else 0)}
    return {"bytes": 2 * B * hkv * case["path"] * token, "flops": 0}


# ---- the same in 64 bits, from the definitions ------------------------------------------


def _attend64(q, k, v, seen=None):
    """[n, 128] queries over [t, 128] keys and values; ``seen`` [n, t] or everything."""
    s = q @ k.T * float(torch.tensor(DIM ** -0.5, dtype=torch.float64).to(torch.float16))
    if seen is not None:
        s.masked_fill_(~seen, -math.inf)
    return torch.softmax(s, -1) @ v


def _exact_prompt(state):
    case = state["case"]
    q, k, v = (state[n].double() for n in ("q", "k", "v"))
    out = torch.zeros_like(q)
    g = case["hq"] // case["hkv"]
    if case["sequences"]:
        starts = _starts(case)
        spans = [(a, b, a, b) for a, b in zip(starts, starts[1:])]
    else:
        spans = [(0, case["tq"], 0, case["tk"])]
    for b in range(case["batch"]):
        for h in range(case["hq"]):
            for q0, q1, k0, k1 in spans:
                for t in range(q0, q1, 4096):
                    end = min(t + 4096, q1)
                    last = k1 - (q1 - end) if case["causal"] else k1  # keys that the last of these queries sees
                    seen = None
                    if case["causal"]:
                        seen = torch.ones((end - t, last - k0), dtype=torch.bool, device="cuda").tril(last - k0 - (end - t))
                    out[b, h, t:end] = _attend64(q[b, h, t:end], k[b, h // g, k0:last], v[b, h // g, k0:last], seen)
    return out


def _decode64(layout, pages, b, h):
    """Keys and values of one (batch, head) in 64 bits."""
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


def _exact_tree(state):
    case = state["case"]
    n, g = case["nodes"], case["hq"] // case["hkv"]
    seen = torch.cat((torch.ones((n, case["tokens"]), dtype=torch.bool, device="cuda"), state["mask"]), 1)
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        for h in range(case["hkv"]):
            keys, values = _decode64(case["layout"], state["pages"], b, h)
            keys = torch.cat((keys, state["tail_k"][b, h].double(), state["k"][b, h].double()))
            values = torch.cat((values, state["tail_v"][b, h].double(), state["v"][b, h].double()))
            for i in range(h * g, (h + 1) * g):
                out[b, i] = _attend64(state["q"][b, i].double(), keys, values, seen)
    return out


def exact(case, seed):
    if case["op"] == "accept":
        return None  # copied, not computed
    if case["op"] == "fork":
        # Copied, but for a tail that is decoded from the page that the prefix ends in.
        S, n, left = case["tokens"] // PAGE, case["keep"] // PAGE, case["keep"] % PAGE
        if not (case["keep"] and n < S and left):
            return None
        state = prepare(case, seed)
        out = {name: None for name in state["pages"]}
        rows = state.get("rows") or range(case["batch"])
        page = {name: t[:, :, n:n + 1] for name, t in state["pages"].items()}
        both = [[_decode64(case["layout"], page, b, h) for h in range(case["hkv"])] for b in rows]
        out["tail.k"] = torch.stack([torch.stack([x[0][:left] for x in row]) for row in both])
        out["tail.v"] = torch.stack([torch.stack([x[1][:left] for x in row]) for row in both])
        return out
    state = prepare(case, seed)
    return _exact_prompt(state) if case["op"] == "prompt" else _exact_tree(state)
