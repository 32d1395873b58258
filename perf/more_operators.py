"""The calls of a decoder's attention block, second part: norms of each head of q and k in the append's own pass, a paged
cache held in 8 bits (int8 or e4m3, a scale for each block of 16 positions and head) that is quantized as it is written and
read back, attention over it, and attention with a window beside which the first positions stay visible.

A case is a dict of plain values; `kind` is "append", "read" or "attend" and `cache` what the pages hold: "same" (the
case's precision), "int8" or "fp8". An append to an 8-bit cache is followed by a read of the blocks that it wrote, so that
the stored values come back as numbers. Lengths of the sequences of a batch are drawn between the case's bounds from its
`lens`. `own` chooses between the plain form (elementary torch operations in 32 bits) and this library's entry points.
"""
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 16                  # positions that share a scale
LEAST = 2.0 ** -64          # no block counts as smaller than this
LARGEST = {"int8": 127.0, "fp8": 448.0}
EPS = 1e-6


def _gie():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-inference_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gie
    return gie


def _case(kind, cache, batch, new, ctx, heads, kv_heads, dim, page, precision, lens, **more):
    """`new` and `ctx`: (least, most) new tokens and tokens already in the cache, for each sequence."""
    case = {"kind": kind, "cache": cache, "batch": batch, "new_least": new[0], "new_most": new[1], "ctx_least": ctx[0],
            "ctx_most": ctx[1], "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "precision": precision, "lens": lens}
    if kind == "append":
        case |= {"rotary": dim, "interleaved": False}
    if kind == "attend":
        case |= {"window": 0, "sinks": 0, "softcap": 0.0}
    return {**case, **more}


def listed():
    cases = {
        # one new token for each of 64 sequences, heads of q and k normed on their way: latency
        "append_norm_step": _case("append", "same", 64, (1, 1), (100, 8000), 32, 8, 128, 16, "fp16", 1),
        # long prompts at once: the bytes
        "append_norm_prompt": _case("append", "same", 2, (4096, 4096), (0, 0), 32, 8, 128, 64, "bf16", 2),
        # a decode step into the 8-bit cache: most blocks hold older tokens, whose scale may have to grow
        "append8_step": _case("append", "int8", 64, (1, 1), (100, 8000), 32, 8, 128, 16, "bf16", 3),
        # chunks of odd lengths into blocks that are partly filled, heads of 96 of which 64 rotate, pairs side by side
        "append8_ragged": _case("append", "fp8", 7, (1, 1500), (0, 1000), 12, 12, 96, 48, "fp16", 4, rotary=64,
                                interleaved=True),
        # a short batch read back: latency
        "read8_ragged": _case("read", "int8", 5, (1, 700), (0, 0), 10, 2, 64, 48, "fp16", 5),
        # one long sequence leaves the 8-bit cache, as for a reader in 16 bits: the bytes
        "read8_long": _case("read", "fp8", 1, (32768, 32768), (0, 0), 32, 8, 128, 64, "bf16", 6),
        # a decode step far past the window of 1024: two short ranges of each sequence's keys
        "sinks_step": _case("attend", "same", 64, (1, 1), (1, 8000), 32, 8, 128, 16, "bf16", 7, window=1024, sinks=4),
        # a prompt whose rows see the first 16 positions and 1000 more
        "sinks_prompt": _case("attend", "same", 1, (8192, 8192), (0, 0), 32, 8, 128, 64, "fp16", 8, window=1000,
                              sinks=16),
        # one token over a long context in 8 bits: the cache's one pass through memory, split over the device
        "attend8_one_long": _case("attend", "int8", 1, (1, 1), (65535, 65535), 32, 8, 128, 64, "bf16", 9),
        # a decode step of 64 sequences of very different lengths over small pages
        "attend8_step_ragged": _case("attend", "fp8", 64, (1, 1), (1, 8000), 32, 8, 128, 16, "fp16", 10),
        # chunks of odd lengths, five heads to a key head, wide heads, a window with sinks, capped scores
        "attend8_ragged_sinks": _case("attend", "int8", 5, (0, 190), (0, 4000), 10, 2, 256, 48, "bf16", 11,
                                      window=1000, sinks=20, softcap=30.0),
        # whole prompts over what was just stored: the most arithmetic
        "attend8_prompt": _case("attend", "int8", 2, (4096, 4096), (0, 0), 32, 8, 128, 64, "bf16", 12),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _draw(rng):
    kind = rng.choice(("append", "append", "read", "attend", "attend", "attend"))
    cache = rng.choice(("int8", "fp8")) if kind == "read" else rng.choice(("same", "int8", "fp8"))
    batch, most_new = rng.choice((1, _log_int(rng, 1, 64))), rng.choice((1, 1, _log_int(rng, 2, 4096)))
    most_ctx = rng.choice((0, _log_int(rng, 1, 65536), _log_int(rng, 1, 65536)))
    if kind == "read":
        most_new, most_ctx = _log_int(rng, 1, 32768), 0
    new = (most_new if rng.random() < 0.5 else rng.randint(0, most_new), most_new)
    ctx = (most_ctx if rng.random() < 0.3 else rng.randint(0, most_ctx), most_ctx)
    kv_heads, group = rng.choice((1, 2, 4, 8, 8, 16)), rng.choice((1, 2, 3, 4, 4, 5, 7, 8))
    dim = rng.choice((64, 96, 128, 128, 256))
    more = {}
    if kind == "append":
        more = {"rotary": rng.choice((dim, dim, dim // 2, 32)), "interleaved": rng.random() < 0.5}
    elif kind == "attend":
        more = {"window": rng.choice((0, 0, _log_int(rng, 64, 4096))), "softcap": rng.choice((0.0, 0.0, 30.0, 50.0))}
        if more["window"] == 0 and cache == "same":
            more["window"] = _log_int(rng, 64, 4096)  # without a window there is nothing that stays visible beside it
        if more["window"]:
            more["sinks"] = rng.choice((1, 4, 16, _log_int(rng, 1, 200)))
    return _case(kind, cache, batch, new, ctx, kv_heads * group, kv_heads, dim, rng.choice((16, 16, 32, 48, 64, 128, 256)),
                 rng.choice(("fp16", "bf16")), rng.randrange(1 << 30), **more)


def _costs(case):
    """What a drawn case may not have more of than the largest listed one: operations, bytes, the cache's values, and
    what the plain form holds at once (scores, gathered keys)."""
    w = work(case)
    new, lengths = _lengths(case)
    pages = sum(-(-n // case["page"]) for n in lengths) + 1
    cache = 2.0 * pages * case["page"] * case["kv_heads"] * case["dim"]
    if case["kind"] != "attend":
        return w["bytes"] / 210e6, cache / 1e9
    # the plain form pads every sequence to the longest
    scores = case["batch"] * case["heads"] * max(new) * float(max(lengths))
    keys = case["batch"] * case["kv_heads"] * float(max(lengths)) * case["dim"]
    return w["flops"] / 276e9, cache / 1e9, scores / 2.2e9, keys / 0.6e9


def draw(rng):
    while True:
        case = _draw(rng)
        if sum(_lengths(case)[0]) > 0 and max(_costs(case)) <= 1.0:
            return case


def _lengths(case):
    """New tokens and total length (the new ones counted) of each sequence; the longest chunk is there at least once."""
    rng = random.Random(case["lens"])
    new = [rng.randint(case["new_least"], case["new_most"]) for _ in range(case["batch"])]
    new[-1] = case["new_most"]
    return new, [n + rng.randint(case["ctx_least"], case["ctx_most"]) for n in new]


def _blocks(case):
    """Rows of the read that follows an append: each sequence from the start of the block of its first new token on."""
    return [n and length - (length - n) // BLOCK * BLOCK for n, length in zip(*_lengths(case))]


def _codes(x, cache):
    """Bytes and scales [pages][heads][page / 16] of values [pages][heads][page][dim], for the cache that a case starts with."""
    blocks = x.reshape(*x.shape[:2], -1, BLOCK, x.shape[3])
    most = blocks.abs().amax((3, 4)).clamp_min(LEAST)
    if cache == "int8":
        scale = most / 127
        codes = (blocks / scale[..., None, None]).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    else:
        scale = torch.exp2(torch.ceil(torch.log2(most / 448)))
        codes = (blocks / scale[..., None, None]).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.reshape(x.shape).contiguous(), scale.contiguous()


def _inputs(case, seed):
    """New q, k, v as a fused projection leaves them (one row for each token), a cache whose pages are scattered and
    hold older values in every slot (blocks of very different size), and the batch's lengths and page table."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new, lengths = _lengths(case)
    heads, kv, dim, page, dtype = case["heads"], case["kv_heads"], case["dim"], case["page"], DTYPES[case["precision"]]
    per_seq = [-(-n // page) for n in lengths]
    max_pages, pages = max(max(per_seq), 1), sum(per_seq) + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
    table, at = torch.zeros((case["batch"], max_pages), dtype=torch.int32), 0
    for b, count in enumerate(per_seq):
        table[b, :count] = order[at:at + count]
        at += count

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    starts = torch.tensor([sum(new[:b]) for b in range(case["batch"] + 1)], dtype=torch.int32)
    d = {"starts": starts.cuda(), "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(), "table": table.cuda()}
    if case["kind"] != "read":
        d["qkv"] = normal(sum(new), (heads + 2 * kv) * dim).to(dtype)
    for n in ("k", "v"):
        values = normal(pages, kv, page, dim)
        if case["cache"] == "same":
            d[n + "_pages"] = values.to(dtype)
        else:
            size = torch.exp(0.5 * normal(pages, kv, page // BLOCK, 1, 1))
            values = (values.reshape(pages, kv, page // BLOCK, BLOCK, dim) * size).reshape(values.shape)
            d[n + "_pages"], d[n + "_scales"] = _codes(values, case["cache"])
    if case["kind"] == "append":
        d["q_norm"], d["k_norm"] = 1 + 0.2 * normal(dim), 1 + 0.2 * normal(dim)
        half = case["rotary"] // 2
        angles = torch.arange(max_pages * page, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(half, device="cuda", dtype=torch.float64) / half)
        d |= {"cos": angles.cos().float(), "sin": angles.sin().float()}
        if case["cache"] != "same":
            rows = _blocks(case)
            d["read_starts"] = torch.tensor([sum(rows[:b]) for b in range(case["batch"] + 1)], dtype=torch.int32).cuda()
    return d


def _split(case, qkv):
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = qkv[:, :heads * dim], qkv[:, heads * dim:(heads + kv) * dim], qkv[:, (heads + kv) * dim:]
    return q, k, v


def prepare(case, seed):
    d = _inputs(case, seed)
    new, lengths = _lengths(case)
    state = {"case": case, "most_new": max(new), "most_len": max(lengths), "tokens": sum(new)} | d
    if "qkv" in d:
        state |= dict(zip("qkv", _split(case, d["qkv"])))
    rows = sum(_blocks(case)) if "read_starts" in d else sum(new)
    state["rows"] = rows
    if own:
        gie, dtype = _gie(), DTYPES[case["precision"]]
        stride = d["qkv"].shape[1] if "qkv" in d else 0
        common = dict(precision=case["precision"], max_new=state["most_new"], max_len=state["most_len"],
                      cache="" if case["cache"] == "same" else case["cache"])
        sizes = (case["heads"], case["kv_heads"], case["dim"], case["page"], d["k_pages"].shape[0], d["table"].shape[1])
        p = gie.PagedKv(case["batch"], sum(new), *sizes, q_stride=stride, k_stride=stride, v_stride=stride,
                        rotary_dim=case.get("rotary", 0), interleaved=case.get("interleaved", False),
                        window=case.get("window", 0), sinks=case.get("sinks", 0), softcap=case.get("softcap", 0.0),
                        max_positions=d["cos"].shape[0] if "cos" in d else 0, norm_eps=EPS, **common)
        state["p"] = p
        if case["kind"] != "read":
            state["out"] = torch.empty((sum(new), case["heads"], case["dim"]), dtype=dtype, device="cuda")
        if case["cache"] != "same" and case["kind"] != "attend":
            state["p_read"] = gie.PagedKv(case["batch"], rows, *sizes, **common)
            for n in ("k_rows", "v_rows"):
                state[n] = torch.empty((rows, case["kv_heads"], case["dim"]), dtype=dtype, device="cuda")
        if case["kind"] == "attend":
            size = gie.paged_attention_workspace_size(p) if case["cache"] == "same" else \
                gie.kv8_attention_workspace_size(p)
            state["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return state


def _positions(starts, lengths, rows):
    """Sequence and position of every row."""
    starts, lengths = starts.long(), lengths.long()
    row = torch.arange(rows, device=starts.device)
    seq = torch.searchsorted(starts, row, right=True) - 1
    return seq, lengths[seq] - starts[seq + 1] + row


def _values(codes, cache):
    return codes.view(torch.int8).float() if cache == "int8" else codes.view(torch.float8_e4m3fn).float()


def _plain_turned(s, position):
    """q, k and v in 32 bits: q and k normed and turned."""
    case, half = s["case"], s["case"]["rotary"] // 2
    cos, sin = s["cos"][position][:, None], s["sin"][position][:, None]

    def turned(x, heads, weight):
        x = x.reshape(x.shape[0], heads, case["dim"]).float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
        y = x.clone()
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else \
            (slice(0, half), slice(half, 2 * half))
        y[..., first] = x[..., first] * cos - x[..., second] * sin
        y[..., second] = x[..., first] * sin + x[..., second] * cos
        return y

    return (turned(s["q"], case["heads"], s["q_norm"]), turned(s["k"], case["kv_heads"], s["k_norm"]),
            s["v"].reshape(-1, case["kv_heads"], case["dim"]).float())


def _plain_append(s):
    case, dtype = s["case"], DTYPES[s["case"]["precision"]]
    seq, position = _positions(s["starts"], s["lengths"], s["tokens"])
    q, k, v = _plain_turned(s, position)
    page, slot = s["table"][seq, position // case["page"]].long(), position % case["page"]
    if case["cache"] == "same":
        s["k_pages"][page, :, slot] = k.to(dtype)
        s["v_pages"][page, :, slot] = v.to(dtype)
        return {"q": q.to(dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    # rows of the blocks that are written: older tokens of a block, then the new ones
    seq, position = _positions(s["read_starts"], s["lengths"], s["rows"])
    first_new = s["lengths"].long()[seq] - (s["starts"][1:] - s["starts"][:-1]).long()[seq]
    fresh = position >= first_new
    token = (s["starts"].long()[seq] + position - first_new).clamp_min(0)
    page, slot = s["table"][seq, position // case["page"]].long(), position % case["page"]
    block = page * (case["page"] // BLOCK) + slot // BLOCK
    part = torch.zeros(s["k_scales"].shape[0] * (case["page"] // BLOCK), device=q.device).index_fill_(0, block[~fresh], 1.0)
    older = part[block] > 0  # the row's block holds older tokens
    out = {"q": q.to(dtype)}
    for name, new in (("k", k), ("v", v)):
        codes, scales = s[name + "_pages"], s[name + "_scales"]
        x = torch.where(fresh[:, None, None], new[token], 0.0)
        most = torch.zeros((part.shape[0], case["kv_heads"]), device=q.device)
        most = most.scatter_reduce(0, block[:, None].expand(-1, case["kv_heads"]), x.abs().amax(2), "amax")
        most = most[block].clamp_min(LEAST)
        if case["cache"] == "int8":
            scale = most / 127
        else:
            mantissa, power = torch.frexp(most)  # 448 = 0.875 2^9
            scale = torch.ldexp(torch.ones_like(most), power - 9 + (mantissa > 0.875))
        before = scales[page, :, slot // BLOCK]
        scale = torch.where(older[:, None], torch.maximum(scale, before), scale)
        y = torch.where(fresh[:, None, None], x, _values(codes[page, :, slot], case["cache"]) * before[..., None])
        y = y / scale[..., None]
        if case["cache"] == "int8":
            y = y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
        else:
            y = y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        codes[page, :, slot] = y
        scales[page, :, slot // BLOCK] = scale
        out[name] = (_values(y, case["cache"]) * scale[..., None]).to(dtype)
    return out


def _plain_read(s):
    case = s["case"]
    seq, position = _positions(s["starts"], s["lengths"], s["rows"])
    page, slot = s["table"][seq, position // case["page"]].long(), position % case["page"]
    return {n: (_values(s[n + "_pages"][page, :, slot], case["cache"]) *
                s[n + "_scales"][page, :, slot // BLOCK][..., None]).to(DTYPES[case["precision"]]) for n in "kv"}


def _plain_attend(s):
    case = s["case"]
    batch, heads, kv, dim = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    group, new, length = heads // kv, s["most_new"], s["most_len"]
    seq, position = _positions(s["starts"], s["lengths"], s["tokens"])
    index = torch.arange(s["tokens"], device=seq.device) - s["starts"].long()[seq]
    q = torch.zeros((batch, new, kv, group, dim), device=seq.device)
    q[seq, index] = s["q"].reshape(-1, kv, group, dim).float()
    q = q.permute(0, 2, 3, 1, 4).reshape(batch * kv, group * new, dim)
    key = torch.arange(length, device=seq.device)
    page, slot = s["table"].long()[:, key // case["page"]], key % case["page"]

    def gather(name):
        x = s[name + "_pages"][page, :, slot]
        if case["cache"] == "same":
            x = x.float()
        else:
            x = _values(x, case["cache"]) * s[name + "_scales"][page, :, slot // BLOCK][..., None]
        return x.permute(0, 2, 1, 3).reshape(batch * kv, length, dim)

    scores = torch.bmm(q, gather("k").transpose(1, 2).contiguous()) * dim ** -0.5
    if case["softcap"] > 0:
        scores = torch.tanh(scores / case["softcap"]) * case["softcap"]
    at = torch.full((batch, new), -1, device=seq.device, dtype=torch.long)
    at[seq, index] = position
    seen = key <= at[:, :, None]
    if case["window"] > 0:
        seen &= (key > at[:, :, None] - case["window"]) | (key < case["sinks"])
    scores = scores.reshape(batch, kv * group, new, length)
    scores = torch.where(seen[:, None], scores, float("-inf"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-3e38))
    weights /= weights.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.bmm(weights.reshape(batch * kv, group * new, length), gather("v"))
    out = out.reshape(batch, kv, group, new, dim)[seq, :, :, index]
    return out.reshape(-1, heads, dim).to(s["q"].dtype)


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[kind](s)
    gie, p = _gie(), s["p"]
    stream = torch.cuda.current_stream().cuda_stream
    where = [s[n].data_ptr() for n in ("starts", "lengths", "table")]
    pages = [s[n].data_ptr() for n in ("k_pages", "v_pages", "k_scales", "v_scales") if n in s]
    if kind == "append":
        call = gie.kv_append_normed if s["case"]["cache"] == "same" else gie.kv8_append
        call(p, s["k"].data_ptr(), s["v"].data_ptr(), *where, *pages, q_norm=s["q_norm"].data_ptr(),
             k_norm=s["k_norm"].data_ptr(), cos=s["cos"].data_ptr(), sin=s["sin"].data_ptr(), q=s["q"].data_ptr(),
             q_out=s["out"].data_ptr(), stream=stream)
        if s["case"]["cache"] == "same":
            return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        where[0] = s["read_starts"].data_ptr()
    if kind != "attend":
        gie.kv8_read(s["p_read"], *pages, *where, s["k_rows"].data_ptr(), s["v_rows"].data_ptr(), stream=stream)
        out = {"k": s["k_rows"], "v": s["v_rows"]}
        return out | {"q": s["out"]} if kind == "append" else out
    call = gie.paged_attention if s["case"]["cache"] == "same" else gie.kv8_attention
    call(p, s["q"].data_ptr(), *pages, *where, s["out"].data_ptr(), workspace=s["workspace"].data_ptr(),
         ws_bytes=s["workspace"].numel(), stream=stream)
    return s["out"]


def work(case):
    new, lengths = _lengths(case)
    tokens, dim, heads, kv = sum(new), case["dim"], case["heads"], case["kv_heads"]
    held = 2 if case["cache"] == "same" else 1 + 4 / (BLOCK * dim)  # bytes of a value in the cache
    if case["kind"] == "read":
        return {"bytes": float(2 * tokens * kv * dim * (2 + held)), "flops": float(2 * tokens * kv * dim)}
    if case["kind"] == "append":
        values = tokens * ((heads + 2 * kv) * dim * 2 + heads * dim * 2 + 2 * kv * dim * held) + tokens * case["rotary"] * 4
        if case["cache"] != "same":
            values += 2 * sum(_blocks(case)) * kv * dim * (2 + held)
        return {"bytes": float(values), "flops": float(tokens * (heads + kv) * (4 * dim + 3 * case["rotary"]))}
    pairs, keys, window, sinks = 0, 0, case["window"], case["sinks"]
    for n, length in zip(new, lengths):
        if n == 0:
            continue
        position = np.arange(length - n, length, dtype=np.int64)
        if window:
            pairs += int((np.minimum(position + 1, window) + np.clip(position + 1 - window, 0, sinks)).sum())
            oldest = max(0, length - n + 1 - window)
            keys += length - oldest + min(oldest, sinks)
        else:
            pairs += int((position + 1).sum())
            keys += length
    return {"bytes": float(2 * tokens * heads * dim * 2 + 2 * keys * kv * dim * held), "flops": 4.0 * dim * heads * pairs}


def _exact_held(case, d, name):
    """Values of the whole cache in 64 bits."""
    codes = d[name + "_pages"]
    if case["cache"] == "same":
        return codes.double()
    if case["cache"] == "int8":
        code = codes.double()
        code = torch.where(code > 127, code - 256, code)
    else:
        bits = codes.to(torch.int64)
        power, fraction = (bits >> 3) & 15, (bits & 7).double()
        code = torch.where(power == 0, fraction / 8 * 2.0 ** -6, (1 + fraction / 8) * torch.exp2((power - 7).double()))
        code = torch.where(bits > 127, -code, code)
    return code * d[name + "_scales"].double().repeat_interleave(BLOCK, dim=2)[..., None]


def _exact_stored(case, x, scale):
    """What x becomes under a scale."""
    y = x / scale
    if case["cache"] == "int8":
        return torch.round(y).clamp(-127, 127) * scale
    power = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(power - 3)
    return (torch.round(y / step) * step).clamp(-448, 448) * scale


def _exact_append(case, seed):
    d = _inputs(case, seed)
    new, lengths = _lengths(case)
    heads, kv, dim, page, half = case["heads"], case["kv_heads"], case["dim"], case["page"], case["rotary"] // 2
    table = d["table"].cpu()
    held = {n: _exact_held(case, d, n) for n in "kv"}
    even = torch.arange(half, device="cuda")
    pairs = torch.stack([2 * even, 2 * even + 1] if case["interleaved"] else [even, even + half])
    queries, rows, start = [], {"k": [], "v": []}, 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        if n == 0:
            continue
        first = length - n
        row = d["qkv"][start:start + n].double().reshape(n, heads + 2 * kv, dim)
        start += n
        both = row[:, :heads + kv]
        both = both / torch.sqrt(both.square().sum(2, keepdim=True) / dim + EPS)
        both = torch.cat([both[:, :heads] * d["q_norm"].double(), both[:, heads:] * d["k_norm"].double()], dim=1)
        cos, sin = d["cos"][first:length].double()[:, None], d["sin"][first:length].double()[:, None]
        turned = both.clone()
        turned[:, :, pairs[0]] = both[:, :, pairs[0]] * cos - both[:, :, pairs[1]] * sin
        turned[:, :, pairs[1]] = both[:, :, pairs[1]] * cos + both[:, :, pairs[0]] * sin
        queries.append(turned[:, :heads])
        fresh = {"k": turned[:, heads:], "v": row[:, heads + kv:]}
        if case["cache"] == "same":
            for j in range(first // page, -(-length // page)):
                lo, hi = max(j * page, first), min((j + 1) * page, length)
                for name in "kv":
                    held[name][int(table[b, j]), :, lo - j * page:hi - j * page] = \
                        fresh[name][lo - first:hi - first].transpose(0, 1)
            continue
        begin = first // BLOCK * BLOCK
        blocks = -(-(length - begin) // BLOCK)
        for name in "kv":
            old_at = torch.arange(begin, first)
            at_page, at_slot = table[b, old_at // page].long().cuda(), (old_at % page).cuda()
            x = torch.cat([held[name][at_page, :, at_slot], fresh[name]])
            pad = torch.zeros((blocks * BLOCK, kv, dim), dtype=torch.float64, device="cuda")
            pad[first - begin:length - begin] = fresh[name]
            most = pad.reshape(blocks, BLOCK, kv, dim).abs().amax((1, 3)).clamp(min=LEAST)
            scale = most / LARGEST[case["cache"]]
            if case["cache"] == "fp8":
                scale = torch.exp2(torch.ceil(torch.log2(scale)))
            if first > begin:
                was = d[name + "_scales"][int(table[b, begin // page]), :, begin % page // BLOCK].double()
                scale[0] = torch.maximum(scale[0], was)
            scale = scale.repeat_interleave(BLOCK, dim=0)[:length - begin, :, None]
            rows[name].append(_exact_stored(case, x, scale))
    q = torch.cat(queries)
    if case["cache"] == "same":
        return {"q": q, "k_pages": held["k"], "v_pages": held["v"]}
    return {"q": q, "k": torch.cat(rows["k"]), "v": torch.cat(rows["v"])}


def _exact_read(case, seed):
    d = _inputs(case, seed)
    out, (new, lengths) = {}, _lengths(case)
    for name in "kv":
        held, rows = _exact_held(case, d, name), []
        for b, (n, length) in enumerate(zip(new, lengths)):
            used = d["table"][b, :-(-length // case["page"])].long()
            rows.append(held[used].transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])[length - n:length])
        out[name] = torch.cat(rows)
    return out


def _exact_attend(case, seed):
    d = _inputs(case, seed)
    new, lengths = _lengths(case)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group, held = heads // kv, {n: _exact_held(case, d, n) for n in "kv"}
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
            hidden |= (key[None, :] <= position[:, None] - case["window"]) & (key[None, :] >= case["sinks"])
        result = torch.empty((n, heads, dim), dtype=torch.float64, device="cuda")
        for h in range(heads):
            k = held["k"][used, h // group].reshape(-1, dim)[:length]
            v = held["v"][used, h // group].reshape(-1, dim)[:length]
            s = (q[:, h] @ k.t().contiguous()) / dim ** 0.5
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            s[hidden] = float("-inf")
            result[:, h] = torch.softmax(s, dim=1) @ v
        out.append(result)
    return torch.cat(out)


def exact(case, seed):
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[case["kind"]](case, seed)
