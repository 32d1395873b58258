"""The calls of a decoder's attention block whose speed this library is held to: the matrix product in 8-bit integers
(scales for each token and output channel, the token's scale found on the way or given), the append of keys and values
to a paged cache with the position rotation, and the attention of the new tokens over that cache. One token for each
sequence, chunks of new tokens and whole prompts; grouped heads, windows and capped scores; odd and ragged sizes.

A case is a dict of plain values; `kind` is "linear", "append" or "attend". Lengths of the sequences of a batch are
drawn between the case's bounds from its `lens`. `own` chooses between the plain form (elementary torch operations in
32 bits) and this library's entry points.
"""
import os
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _gie():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-inference_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gie
    return gie


def _linear(m, k, n, precision, bias=False, relu=False, quantized=False):
    return {"kind": "linear", "m": m, "k": k, "n": n, "precision": precision, "bias": bias, "relu": relu,
            "quantized": quantized}


def _paged(kind, batch, new, ctx, heads, kv_heads, dim, page, precision, lens, **more):
    """`new` and `ctx`: (least, most) new tokens and tokens already in the cache, for each sequence."""
    case = {"kind": kind, "batch": batch, "new_least": new[0], "new_most": new[1], "ctx_least": ctx[0],
            "ctx_most": ctx[1], "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "precision": precision, "lens": lens}
    if kind == "append":
        case |= {"rotary": dim, "interleaved": False}
    else:
        case |= {"window": 0, "softcap": 0.0}
    return {**case, **more}


def listed():
    cases = {
        # the projection of one token of one sequence: latency, and the weights' one pass through memory
        "linear_one_token": _linear(1, 4096, 4096, "fp16"),
        # a decode step of 64 sequences: still bound by the weights
        "linear_64_tokens": _linear(64, 8192, 8192, "bf16", relu=True),
        # odd extents everywhere, activations already in 8 bits, 32-bit result with its bias
        "linear_ragged_fp32": _linear(77, 1000, 2050, "fp32", bias=True, quantized=True),
        # the widest projection of a long prompt: the most arithmetic
        "linear_prompt": _linear(4096, 4096, 16384, "fp16", bias=True),
        # one new token for each of 64 sequences
        "append_step": _paged("append", 64, (1, 1), (100, 8000), 32, 8, 128, 16, "fp16", 1),
        # chunks of odd lengths, heads of 96 of which 64 rotate, pairs side by side, pages of 48
        "append_ragged": _paged("append", 7, (1, 333), (0, 1000), 12, 12, 96, 48, "bf16", 2, rotary=64,
                                interleaved=True),
        # a long prompt goes into the cache at once
        "append_prompt": _paged("append", 2, (4096, 4096), (0, 0), 32, 8, 128, 64, "bf16", 3),
        # one sequence with a long context, one new token: the cache's one pass through memory, split over the device
        "attend_one_long": _paged("attend", 1, (1, 1), (32767, 32767), 32, 8, 128, 64, "bf16", 4),
        # a decode step of 64 sequences of very different lengths over small pages
        "attend_step_ragged": _paged("attend", 64, (1, 1), (1, 8000), 32, 8, 128, 16, "fp16", 5),
        # a chunk of a prompt over what the cache already holds
        "attend_chunk": _paged("attend", 1, (512, 512), (7680, 7680), 32, 8, 128, 64, "fp16", 6),
        # chunks of odd lengths, five heads to a key head, a window and capped scores, wide heads
        "attend_ragged_window": _paged("attend", 5, (0, 190), (0, 3000), 10, 2, 256, 48, "bf16", 7, window=1000,
                                       softcap=30.0),
        # whole prompts, nothing in the cache before: the most arithmetic of the attention
        "attend_prompt": _paged("attend", 2, (4096, 4096), (0, 0), 32, 8, 128, 64, "bf16", 8),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _features(rng, lo, hi):
    """Mostly multiples of 128, some of 8, some of nothing."""
    v, r = _log_int(rng, lo, hi), rng.random()
    v = v if r < 0.2 else max(8, v // 8 * 8) if r < 0.4 else max(128, v // 128 * 128)
    return v + 128 if v == 3072 else v


def _draw(rng):
    kind = rng.choice(("linear", "append", "attend"))
    if kind == "linear":
        return _linear(_log_int(rng, 1, 8192), _features(rng, 64, 16384), _features(rng, 64, 16384),
                       rng.choice(("fp16", "bf16", "fp16", "bf16", "fp32")), rng.random() < 0.5, rng.random() < 0.3,
                       rng.random() < 0.4)
    batch, most_new = rng.choice((1, _log_int(rng, 1, 64))), rng.choice((1, 1, _log_int(rng, 2, 4096)))
    most_ctx = rng.choice((0, _log_int(rng, 1, 32768), _log_int(rng, 1, 32768)))
    new = (most_new if rng.random() < 0.5 else rng.randint(0, most_new), most_new)
    ctx = (most_ctx if rng.random() < 0.3 else rng.randint(0, most_ctx), most_ctx)
    kv_heads, group = rng.choice((1, 2, 4, 8, 8, 16)), rng.choice((1, 2, 3, 4, 4, 5, 7, 8))
    dim = rng.choice((64, 96, 128, 128, 256))
    more = {}
    if kind == "append":
        more = {"rotary": rng.choice((dim, dim, dim // 2, 32)), "interleaved": rng.random() < 0.5}
    else:
        more = {"window": rng.choice((0, 0, 0, _log_int(rng, 64, 4096))), "softcap": rng.choice((0.0, 0.0, 30.0, 50.0))}
    return _paged(kind, batch, new, ctx, kv_heads * group, kv_heads, dim, rng.choice((16, 16, 32, 48, 64, 128, 256)),
                  rng.choice(("fp16", "bf16")), rng.randrange(1 << 30), **more)


def _costs(case):
    """What a drawn case may not have more of than the largest listed one: operations, the cache's bytes, and the
    values that the plain form holds at once (scores, gathered keys)."""
    w = work(case)
    if case["kind"] == "linear":
        return w["flops"] / (2 * 4096 * 4096 * 16384), w["bytes"] / 300e6
    new, lengths = _lengths(case)
    pages = sum(-(-n // case["page"]) for n in lengths) + 1
    cache = 2.0 * pages * case["page"] * case["kv_heads"] * case["dim"] * 2
    if case["kind"] == "append":
        return w["bytes"] / 210e6, cache / 2e9
    # the plain form pads every sequence to the longest
    scores = case["batch"] * case["heads"] * max(new) * float(max(lengths))
    keys = case["batch"] * case["kv_heads"] * float(max(lengths)) * case["dim"]
    return w["flops"] / 276e9, cache / 2e9, scores / 1.1e9, keys / 0.6e9


def draw(rng):
    while True:
        case = _draw(rng)
        if case["kind"] != "linear" and (sum(_lengths(case)[0]) == 0):
            continue
        if max(_costs(case)) <= 1.0:
            return case


def _lengths(case):
    """New tokens and total length (the new ones counted) of each sequence; the longest chunk is there at least once."""
    rng = random.Random(case["lens"])
    new = [rng.randint(case["new_least"], case["new_most"]) for _ in range(case["batch"])]
    new[-1] = case["new_most"]
    return new, [n + rng.randint(case["ctx_least"], case["ctx_most"]) for n in new]


def _linear_inputs(case, seed):
    """Activations normal with a few channels ten times as large, weights normal; in 8 bits with one scale a row."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, k, n, dtype = case["m"], case["k"], case["n"], DTYPES[case["precision"]]
    x = torch.randn((m, k), generator=gen, device="cuda")
    x *= 1 + 9 * (torch.rand((k,), generator=gen, device="cuda") < 0.01)
    x_scale = None
    if case["quantized"]:
        x_scale = x.abs().amax(1) / 127
        x = torch.round(x / x_scale[:, None]).to(torch.int8)
    else:
        x = x.to(dtype)
    w = torch.randn((n, k), generator=gen, device="cuda").mul_(30).round_().clamp_(-127, 127).to(torch.int8)
    w_scale = (torch.rand((n,), generator=gen, device="cuda") + 0.5) / (30 * k ** 0.5)
    bias = (torch.rand((n,), generator=gen, device="cuda") - 0.5).to(dtype) if case["bias"] else None
    return x, x_scale, w, w_scale, bias


def _paged_inputs(case, seed):
    """New q, k, v as a fused projection leaves them (one row for each token), a cache whose pages are scattered and
    hold older values in every slot, and the batch's lengths and page table."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new, lengths = _lengths(case)
    heads, kv, dim, page, dtype = case["heads"], case["kv_heads"], case["dim"], case["page"], DTYPES[case["precision"]]
    per_seq = [-(-n // page) for n in lengths]
    max_pages, pages = max(per_seq), sum(per_seq) + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
    table, at = torch.zeros((case["batch"], max_pages), dtype=torch.int32), 0
    for b, count in enumerate(per_seq):
        table[b, :count] = order[at:at + count]
        at += count

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    starts = torch.tensor([sum(new[:b]) for b in range(case["batch"] + 1)], dtype=torch.int32)
    d = {"qkv": normal(sum(new), (heads + 2 * kv) * dim), "k_pages": normal(pages, kv, page, dim),
         "v_pages": normal(pages, kv, page, dim), "starts": starts.cuda(),
         "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(), "table": table.cuda()}
    if case["kind"] == "append":
        half = case["rotary"] // 2
        angles = torch.arange(max_pages * page, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(half, device="cuda", dtype=torch.float64) / half)
        d |= {"cos": angles.cos().float(), "sin": angles.sin().float()}
    return d


def _split(case, qkv):
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = qkv[:, :heads * dim], qkv[:, heads * dim:(heads + kv) * dim], qkv[:, (heads + kv) * dim:]
    return q, k, v


def prepare(case, seed):
    state = {"case": case}
    if case["kind"] == "linear":
        x, x_scale, w, w_scale, bias = _linear_inputs(case, seed)
        state |= {"x": x, "x_scale": x_scale, "w": w, "w_scale": w_scale, "bias": bias}
        if own:
            gie = _gie()
            p = gie.LinearI8(case["m"], case["k"], case["n"], precision=case["precision"], has_bias=case["bias"],
                             relu=case["relu"], quantized=case["quantized"])
            state |= {"p": p, "y": torch.empty((case["m"], case["n"]), dtype=DTYPES[case["precision"]], device="cuda"),
                      "workspace": torch.empty(gie.linear_i8_workspace_size(p), dtype=torch.uint8, device="cuda")}
        return state
    d = _paged_inputs(case, seed)
    q, k, v = _split(case, d["qkv"])
    state |= d | {"q": q, "k": k, "v": v, "most_new": max(_lengths(case)[0]), "most_len": max(_lengths(case)[1])}
    if own:
        gie = _gie()
        row = d["qkv"].shape[1]
        p = gie.PagedKv(case["batch"], q.shape[0], case["heads"], case["kv_heads"], case["dim"], case["page"],
                        d["k_pages"].shape[0], d["table"].shape[1], precision=case["precision"], q_stride=row,
                        k_stride=row, v_stride=row, rotary_dim=case.get("rotary", 0),
                        interleaved=case.get("interleaved", False), window=case.get("window", 0),
                        softcap=case.get("softcap", 0.0), max_new=state["most_new"], max_len=state["most_len"],
                        max_positions=d["cos"].shape[0] if "cos" in d else 0)
        state |= {"p": p, "out": torch.empty((q.shape[0], case["heads"], case["dim"]), dtype=q.dtype, device="cuda")}
        if case["kind"] == "attend":
            state["workspace"] = torch.empty(gie.paged_attention_workspace_size(p), dtype=torch.uint8, device="cuda")
    return state


def _plain_linear(s):
    x, scale = s["x"].float(), s["x_scale"]
    if scale is None:
        most = x.abs().amax(1).clamp_min(2.0 ** -100)
        scale = most / 127
        x = torch.round(x * (127 / most)[:, None])
    y = x @ s["w"].float().t()
    y = y * scale[:, None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["relu"]:
        y = y.clamp_min(0)
    return y.to(DTYPES[s["case"]["precision"]])


def _positions(s):
    """Sequence and position of every new token."""
    starts, lengths = s["starts"].long(), s["lengths"].long()
    token = torch.arange(s["q"].shape[0], device=starts.device)
    seq = torch.searchsorted(starts, token, right=True) - 1
    return seq, lengths[seq] - starts[seq + 1] + token


def _plain_append(s):
    case = s["case"]
    seq, position = _positions(s)
    half = case["rotary"] // 2
    cos, sin = s["cos"][position][:, None], s["sin"][position][:, None]

    def rotate(x, heads):
        x = x.reshape(x.shape[0], heads, case["dim"]).float()
        y = x.clone()
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else \
            (slice(0, half), slice(half, 2 * half))
        y[..., first] = x[..., first] * cos - x[..., second] * sin
        y[..., second] = x[..., first] * sin + x[..., second] * cos
        return y.to(s["q"].dtype)

    page, slot = s["table"][seq, position // case["page"]].long(), position % case["page"]
    s["k_pages"][page, :, slot] = rotate(s["k"], case["kv_heads"])
    s["v_pages"][page, :, slot] = s["v"].reshape(-1, case["kv_heads"], case["dim"])
    return {"q": rotate(s["q"], case["heads"]), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attend(s):
    case = s["case"]
    batch, heads, kv, dim = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    group, new, length = heads // kv, s["most_new"], s["most_len"]
    seq, position = _positions(s)
    index = torch.arange(s["q"].shape[0], device=seq.device) - s["starts"].long()[seq]
    q = torch.zeros((batch, new, kv, group, dim), device=seq.device)
    q[seq, index] = s["q"].reshape(-1, kv, group, dim).float()
    q = q.permute(0, 2, 3, 1, 4).reshape(batch * kv, group * new, dim)
    key = torch.arange(length, device=seq.device)
    page = s["table"].long()[:, key // case["page"]]

    def gather(pages):
        return pages[page, :, key % case["page"]].float().permute(0, 2, 1, 3).reshape(batch * kv, length, dim)

    scores = torch.bmm(q, gather(s["k_pages"]).transpose(1, 2).contiguous()) * dim ** -0.5
    if case["softcap"] > 0:
        scores = torch.tanh(scores / case["softcap"]) * case["softcap"]
    at = torch.full((batch, new), -1, device=seq.device, dtype=torch.long)
    at[seq, index] = position
    seen = key <= at[:, :, None]
    if case["window"] > 0:
        seen &= key > at[:, :, None] - case["window"]
    scores = scores.reshape(batch, kv * group, new, length)
    scores = torch.where(seen[:, None], scores, float("-inf"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-3e38))
    weights /= weights.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.bmm(weights.reshape(batch * kv, group * new, length), gather(s["v_pages"]))
    out = out.reshape(batch, kv, group, new, dim)[seq, :, :, index]
    return out.reshape(-1, heads, dim).to(s["q"].dtype)


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}[kind](state)
    gie, p, s = _gie(), state["p"], state
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "linear":
        gie.linear_i8(p, s["x"].data_ptr(), s["w"].data_ptr(), s["w_scale"].data_ptr(), s["y"].data_ptr(),
                      x_scale=s["x_scale"].data_ptr() if s["x_scale"] is not None else None,
                      bias=s["bias"].data_ptr() if s["bias"] is not None else None,
                      workspace=s["workspace"].data_ptr(), ws_bytes=s["workspace"].numel(), stream=stream)
        return s["y"]
    if kind == "append":
        gie.kv_append(p, s["k"].data_ptr(), s["v"].data_ptr(), s["starts"].data_ptr(), s["lengths"].data_ptr(),
                      s["table"].data_ptr(), s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), cos=s["cos"].data_ptr(),
                      sin=s["sin"].data_ptr(), q=s["q"].data_ptr(), q_out=s["out"].data_ptr(), stream=stream)
        return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    gie.paged_attention(p, s["q"].data_ptr(), s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["starts"].data_ptr(),
                        s["lengths"].data_ptr(), s["table"].data_ptr(), s["out"].data_ptr(),
                        workspace=s["workspace"].data_ptr(), ws_bytes=s["workspace"].numel(), stream=stream)
    return s["out"]


def work(case):
    size = BYTES[case["precision"]]
    if case["kind"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        values = m * k * (1 if case["quantized"] else size) + n * k + m * n * size + 4 * n
        values += 4 * m * case["quantized"] + n * size * case["bias"]
        return {"bytes": float(values), "flops": 2.0 * m * k * n}
    new, lengths = _lengths(case)
    tokens, dim, heads, kv = sum(new), case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        values = 2 * tokens * (heads + 2 * kv) * dim * size + tokens * case["rotary"] * 4
        return {"bytes": float(values), "flops": 3.0 * tokens * (heads + kv) * case["rotary"]}
    pairs, keys, window = 0, 0, case["window"]
    for n, length in zip(new, lengths):
        first = length - n
        pairs += n * first + n * (n + 1) // 2
        keys += length if n else 0
        if window and n:
            over = [max(0, p + 1 - window) for p in (first, length - 1)]
            # keys that the window takes from each of the n rows: 0 up to position window - 1, then one more each row
            pairs -= (over[0] + over[1]) * (over[1] - over[0] + 1) // 2 if over[0] else over[1] * (over[1] + 1) // 2
            keys -= over[0]
    return {"bytes": float(2 * tokens * heads * dim * size + 2 * keys * kv * dim * size),
            "flops": 4.0 * dim * heads * pairs}


def _exact_linear(case, seed):
    x, x_scale, w, w_scale, bias = _linear_inputs(case, seed)
    x, w = x.double(), w.double()
    if x_scale is None:
        x_scale = x.abs().max(1).values.clamp(min=2.0 ** -100) / 127
        x = torch.round(x / x_scale[:, None])
    y = torch.matmul(x, w.t().contiguous()) * (x_scale.double()[:, None] * w_scale.double()[None, :])
    if bias is not None:
        y += bias.double()
    return y.clamp(min=0) if case["relu"] else y


def _exact_append(case, seed):
    d = _paged_inputs(case, seed)
    new, lengths = _lengths(case)
    heads, kv, dim, page, half = case["heads"], case["kv_heads"], case["dim"], case["page"], case["rotary"] // 2
    k_pages, v_pages = d["k_pages"].double(), d["v_pages"].double()
    table, rows = d["table"].cpu(), []
    even = torch.arange(half, device="cuda")
    pairs = torch.stack([2 * even, 2 * even + 1] if case["interleaved"] else [even, even + half])
    start = 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        row = d["qkv"][start:start + n].double().reshape(n, heads + 2 * kv, dim)
        start += n
        cos, sin = d["cos"][length - n:length].double()[:, None], d["sin"][length - n:length].double()[:, None]
        turned = row.clone()
        u, v = row[:, :heads + kv, pairs[0]], row[:, :heads + kv, pairs[1]]
        turned[:, :heads + kv, pairs[0]] = u * cos - v * sin
        turned[:, :heads + kv, pairs[1]] = v * cos + u * sin
        rows.append(turned[:, :heads])
        for first in range((length - n) // page, -(-length // page)):
            lo, hi = max(first * page, length - n), min((first + 1) * page, length)
            if lo < hi:
                part = turned[lo - (length - n):hi - (length - n)].transpose(0, 1)
                at = int(table[b, first])
                k_pages[at, :, lo - first * page:hi - first * page] = part[heads:heads + kv]
                v_pages[at, :, lo - first * page:hi - first * page] = part[heads + kv:]
    return {"q": torch.cat(rows), "k_pages": k_pages, "v_pages": v_pages}


def _exact_attend(case, seed):
    d = _paged_inputs(case, seed)
    new, lengths = _lengths(case)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = heads // kv
    out, start = [], 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        q = _split(case, d["qkv"][start:start + n])[0].double().reshape(n, heads, dim)
        start += n
        if n == 0:
            continue
        used = d["table"][b, :-(-length // page)].long()
        position = torch.arange(length - n, length, device="cuda")
        key = torch.arange(length, device="cuda")
        hidden = key[None, :] > position[:, None]
        if case["window"]:
            hidden |= key[None, :] <= position[:, None] - case["window"]
        result = torch.empty((n, heads, dim), dtype=torch.float64, device="cuda")
        for h in range(heads):
            k = d["k_pages"][used, h // group].double().reshape(-1, dim)[:length]
            v = d["v_pages"][used, h // group].double().reshape(-1, dim)[:length]
            s = (q[:, h] @ k.t().contiguous()) / dim ** 0.5
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            s[hidden] = float("-inf")
            result[:, h] = torch.softmax(s, dim=1) @ v
        out.append(result)
    return torch.cat(out)


def exact(case, seed):
    return {"linear": _exact_linear, "append": _exact_append, "attend": _exact_attend}[case["kind"]](case, seed)
