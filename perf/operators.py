"""Performance cases of the 8-bit KV cache's operators.

A serving program holds its keys and values in 8 bits (``SwitchKVCache``: e4m3
or int8 codes ``[B, L, Hkv, 128]``, one fp32 scale for each block of tokens and
KV head, ``[B, Hkv, ceil(L / block)]``) and, to keep long sequences inside a
budget, sums up how much attention every key has received:

* ``append``: new bf16 rows, of a prompt or of one token, are quantised into
  the cache (``switch_kv_cache_append``) and read back
  (``switch_kv_cache_read``) from the first block that they touched, as a
  program does that attends what its cache holds.
* ``read``: a range of cached rows as bf16, for a prefill over earlier chunks
  (``switch_kv_cache_read``).
* ``decode``: one routed decode step over the cache
  (``switch_gqa_decode_quantized_forward``), in some cases adding each key's
  attention weight to the running sums.
* ``weights``: the attention weight that each key received from a whole
  prompt's queries (``switch_gqa_prefill_key_weights``).
* ``evict``: the heaviest keys and the newest ones move into a smaller cache
  (``switch_kv_cache_evict``), which is read back.

Scales are powers of two, the smallest that hold a block's largest magnitude,
so that codes and values are the same however they are computed.  head_dim is
128 throughout.  Sizes come from ``switchattentionkernels_amd/workloads.py``
and ``bench.py`` or are generic.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

D = 128
QMAX = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MIN_EXP = -100          # no scale is below 2^-100


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _append(dtype, batch, lo, hi, heads_kv, capacity, block, packed):
    """``lo`` to ``hi`` new rows per sequence, packed (``cu_seqlens``) or padded
    (then every sequence takes ``hi``)."""
    return {"op": "append", "dtype": dtype, "batch": batch, "lo": lo, "hi": hi,
            "heads_kv": heads_kv, "capacity": capacity, "block": block, "packed": packed}


def _read(dtype, batch, rows, heads_kv, capacity, block):
    return {"op": "read", "dtype": dtype, "batch": batch, "rows": rows, "heads_kv": heads_kv,
            "capacity": capacity, "block": block}


def _decode(dtype, batch, capacity, heads_q, heads_kv, window, p_full, block, weights):
    return {"op": "decode", "dtype": dtype, "batch": batch, "capacity": capacity,
            "heads_q": heads_q, "heads_kv": heads_kv, "window": window, "p_full": p_full,
            "block": block, "weights": weights}


def _weights(batch, seq, heads_q, heads_kv, window, p_full):
    return {"op": "weights", "batch": batch, "seq": seq, "heads_q": heads_q, "heads_kv": heads_kv,
            "window": window, "p_full": p_full}


def _evict(dtype, batch, capacity, heads_kv, budget, recent, block):
    return {"op": "evict", "dtype": dtype, "batch": batch, "capacity": capacity,
            "heads_kv": heads_kv, "budget": budget, "recent": recent, "block": block}


def listed():
    return [
        # One decode step's new token of a serving batch: latency only.
        dict(_append("e4m3", 64, 1, 1, 8, 8192, 64, False), name="append_token_b64"),
        # Continuous batching: the packed prompts of eight requests, mixed lengths.
        dict(_append("int8", 8, 512, 8192, 8, 8400, 64, True), name="append_varlen_b8"),
        # A few ragged rows of several requests: the smallest read.
        dict(_read("int8", 8, 199, 8, 4096, 32), name="read_ragged_b8"),
        # The history of a long document, for its next chunk's prefill.
        dict(_read("e4m3", 1, 16384, 8, 16384, 64), name="read_s16k"),
        # One user's decode step: the smallest, latency only.
        dict(_decode("e4m3", 1, 4096, 32, 8, 1024, 1.0, 64, False), name="decode_b1_l4096"),
        # A serving batch in decode: mixed cache lengths and routes.
        dict(_decode("e4m3", 64, 8192, 32, 8, 1024, 0.25, 64, False), name="decode_b64_l8192"),
        # A ragged batch that keeps the sums an eviction needs, five query heads
        # per KV head, half of the tokens routed full.
        dict(_decode("int8", 24, 2999, 40, 8, 512, 0.5, 32, True), name="decode_sums_b24_l2999"),
        # Long documents, all routed full, eight query heads per KV head.
        dict(_decode("int8", 16, 32768, 64, 8, 4096, 1.0, 64, False), name="decode_b16_l32k"),
        # The sums of a short prompt on a small layer.
        dict(_weights(1, 1024, 8, 2, 256, 0.25), name="weights_s1024"),
        # The sums of a long prompt, the benchmark's shape: the largest.
        dict(_weights(1, 16384, 32, 8, 1024, 0.25), name="weights_s16k"),
        # A batch in decode goes back to its budget; some sequences are below it.
        dict(_evict("int8", 32, 4096, 8, 2047, 256, 32), name="evict_b32_l4096"),
        # A long prompt is cut to a quarter before its first decode step.
        dict(_evict("e4m3", 1, 16384, 8, 4096, 1024, 64), name="evict_s16k"),
    ]


_HEADS = [(8, 2), (32, 8), (40, 8), (64, 8), (4, 1)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    """One more case of the listed ones' ranges."""
    op = rng.choice(["append", "read", "decode", "decode", "weights", "evict"])
    heads_q, heads_kv = rng.choice(_HEADS)
    dtype, block = rng.choice(["e4m3", "int8"]), rng.choice([16, 32, 64, 64, 128])
    if op == "append":
        if rng.random() < 0.5:
            return _append(dtype, _log_int(rng, 1, 64), 1, 1, heads_kv, _log_int(rng, 1024, 8192),
                           block, False)
        hi = _log_int(rng, 64, 8192)
        return _append(dtype, rng.randint(1, 8), max(1, hi // 16), hi, heads_kv,
                       hi + rng.randint(0, 300), block, rng.random() < 0.5)
    if op == "read":
        batch = _log_int(rng, 1, 16)
        capacity = _log_int(rng, 512, max(512, 32768 // batch))
        return _read(dtype, batch, _log_int(rng, 64, capacity), heads_kv, capacity, block)
    if op == "decode":
        batch = _log_int(rng, 1, 64)
        return _decode(dtype, batch, _log_int(rng, 512, min(32768, 64 * 8192 // batch)), heads_q,
                       heads_kv, _log_int(rng, 256, 4096), rng.choice([0.0, 0.25, 0.5, 1.0]), block,
                       rng.random() < 0.4)
    if op == "weights":
        batch = rng.choice([1, 1, 2])
        return _weights(batch, _log_int(rng, 512, 16384 // batch if heads_q <= 32 else 8192 // batch),
                        heads_q, heads_kv, _log_int(rng, 256, 4096), round(rng.uniform(0.1, 0.5), 2))
    batch = _log_int(rng, 1, 32)
    capacity = _log_int(rng, 512, min(16384, 32 * 4096 // batch))
    budget = _log_int(rng, capacity // 8, capacity // 2)
    return _evict(dtype, batch, capacity, heads_kv, budget, rng.randint(0, budget // 2), block)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _spread(lo, hi, n):
    """n lengths from lo to hi in equal steps (the longest alone for n = 1)."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _old_lens(case):
    """Rows that the cache holds before an append: none to what still fits."""
    room = case["capacity"] - case["hi"]
    return _spread(min(room, case["capacity"] // 2) if case["hi"] == 1 else 0, room, case["batch"])


def _new_rows(case):
    return _spread(case["lo"], case["hi"], case["batch"])[::-1] if case["packed"] else [case["hi"]] * case["batch"]


def _decode_lens(case):
    return _spread(max(1, case["capacity"] // 2), case["capacity"], case["batch"])


def _decode_full(case):
    p = case["p_full"]
    return [math.floor((i + 1) * p) > math.floor(i * p) if p < 1 else True
            for i in range(case["batch"])]


def _evict_lens(case):
    return _spread(max(1, case["capacity"] // 4), case["capacity"], case["batch"])


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows(gen, *shape):
    """bf16 keys or values: normal, with tokens of different magnitude (a factor
    of about two either way), as the sink and separator tokens of real layers."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    size = torch.exp(0.35 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))
    return (x * size).to(torch.bfloat16)


def _need(amax, dtype):
    """The smallest power of two, at least 2^MIN_EXP, with amax <= QMAX * scale."""
    m, e = torch.frexp(amax)
    top, top_e = math.frexp(QMAX[dtype])
    e = (e - top_e + (m > top)).clamp(min=MIN_EXP)
    e = torch.where(amax > 0, e, MIN_EXP).to(torch.int32)
    return ((e + 127) << 23).view(torch.float32)


def _codes(x, dtype):
    """fp32 values, scaled into the code's range, rounded to codes."""
    return x.to(torch.float8_e4m3fn) if dtype == "e4m3" else torch.round(x).to(torch.int8)


def _cache(gen, case):
    """A cache with every row filled (codes, scales)."""
    b, n, h, blk = case["batch"], case["capacity"], case["heads_kv"], case["block"]
    nblk = -(-n // blk)
    x = _rows(gen, b, nblk * blk, h, D).float().view(b, nblk, blk, h, D)
    scale = _need(x.abs().amax(dim=(2, 4)), case["dtype"])            # [b, nblk, h]
    codes = _codes(x / scale[:, :, None, :, None], case["dtype"]).view(b, nblk * blk, h, D)
    return codes[:, :n].contiguous(), scale.transpose(1, 2).contiguous()


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen, order = _gen(seed), random.Random(int(seed))
    s = {"case": dict(case)}
    if case["op"] == "weights":
        b, n, hq, hkv = case["batch"], case["seq"], case["heads_q"], case["heads_kv"]
        s["q"] = torch.randn(b, n, hq, D, generator=gen, device="cuda").to(torch.bfloat16)
        s["k"] = torch.randn(b, n, hkv, D, generator=gen, device="cuda").to(torch.bfloat16)
        mask = (torch.rand(b, n, generator=gen, device="cuda") < case["p_full"]).view(-1)
        at = torch.arange(b * n, dtype=torch.int32, device="cuda")
        s["full"], s["local"] = at[mask], at[~mask]
        s["lse"] = _prompt_lse(s)
        return s
    perm = list(range(case["batch"]))
    order.shuffle(perm)
    pick = lambda values: [values[i] for i in perm]  # noqa: E731
    s["k"], s["k_scales"] = _cache(gen, case)
    s["v"], s["v_scales"] = _cache(gen, case)
    b, hkv = case["batch"], case["heads_kv"]
    if case["op"] == "append":
        lens, rows = pick(_old_lens(case)), pick(_new_rows(case))
        s["lens"] = _int32(lens)
        s["starts"] = _int32([x // case["block"] * case["block"] for x in lens])
        s["cu"] = [0]
        for x in rows:
            s["cu"].append(s["cu"][-1] + x)
        shape = (1, s["cu"][-1]) if case["packed"] else (b, case["hi"])
        s["new_k"], s["new_v"] = _rows(gen, *shape, hkv, D), _rows(gen, *shape, hkv, D)
    elif case["op"] == "read":
        s["starts"] = _int32(pick(_spread(0, case["capacity"] - case["rows"], b)) if b > 1 else [0])
    elif case["op"] == "decode":
        s["q"] = torch.randn(b, 1, case["heads_q"], D, generator=gen, device="cuda").to(torch.bfloat16)
        s["lens"] = _int32(pick(_decode_lens(case)))
        s["full"] = torch.tensor(pick(_decode_full(case)), device="cuda")
        if case["weights"]:
            s["sums"] = torch.rand(b, hkv, case["capacity"], generator=gen, device="cuda")
    else:
        s["lens"] = _int32(pick(_evict_lens(case)))
        # Attention sums are heavy-tailed; keys of the last steps may have none yet.
        w = torch.exp(2.0 * torch.randn(b, hkv, case["capacity"], generator=gen, device="cuda"))
        s["sums"] = w * (torch.rand(w.shape, generator=gen, device="cuda") > 0.05)
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _visible(case, full):
    """[b, i, j]: whether query i of sequence b sees key j."""
    b, n = case["batch"], case["seq"]
    first = (torch.arange(n, device="cuda") - case["window"] + 1).expand(b, n).clone()
    first.view(-1)[full.long()] = 0
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")
    return (j <= i) & (j >= first[:, :, None])


def _prompt_lse(s):
    """log2 of each query's softmax sum, as the forward leaves it (heads one by
    one, so that the input fits beside anything)."""
    case = s["case"]
    b, n, hq, hkv = case["batch"], case["seq"], case["heads_q"], case["heads_kv"]
    hide = ~_visible(case, s["full"])
    c = D ** -0.5 * math.log2(math.e)
    lse = torch.empty(b, n, hq, device="cuda")
    for h in range(hq):
        kt = s["k"][:, :, h // (hq // hkv)].float().transpose(1, 2).contiguous()
        x = torch.matmul(s["q"][:, :, h].float(), kt).mul_(c * math.log(2)).masked_fill_(hide, -math.inf)
        lse[:, :, h] = torch.logsumexp(x, dim=-1) * math.log2(math.e)
    return lse


def _plain_weights(s):
    case = s["case"]
    b, n, hq, hkv = case["batch"], case["seq"], case["heads_q"], case["heads_kv"]
    g, c = hq // hkv, D ** -0.5 * math.log2(math.e)
    q = s["q"].float().view(b, n, hkv, g, D).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * n, D)
    kt = s["k"].float().permute(0, 2, 3, 1).contiguous()
    x = torch.matmul(q, kt).view(b, hkv, g, n, n).mul_(c)
    x.sub_(s["lse"].view(b, n, hkv, g).permute(0, 2, 3, 1)[..., None]).exp2_()
    x.masked_fill_(~_visible(case, s["full"])[:, None, None], 0.0)
    return x.sum(dim=(2, 3))


def _values(codes, scales, block):
    """fp32 [B, L, Hkv, 128] of a whole cache."""
    n = codes.shape[1]
    per_row = scales.transpose(1, 2).repeat_interleave(block, dim=1)[:, :n]
    return codes.float() * per_row[..., None]


def _plain_rows(codes, scales, block, starts, rows, lens):
    """bf16 [B, rows, Hkv, 128] from row starts[b] on; 0 from lens[b] on."""
    n = codes.shape[1]
    at = starts.long()[:, None] + torch.arange(rows, device="cuda")
    end = torch.full_like(starts, n) if lens is None else lens
    live = at < end.long()[:, None]
    at = at.clamp(max=n - 1)
    b = torch.arange(codes.shape[0], device="cuda")[:, None]
    x = codes.view(torch.uint8)[b, at].view(codes.dtype).float()
    x = x * scales.transpose(1, 2)[b, at // block][..., None]
    return torch.where(live[:, :, None, None], x, 0.0).to(torch.bfloat16)


def _plain_store(codes, scales, new, seq, at, lens, case):
    """Quantise rows new [N, Hkv, 128] into rows at of sequences seq."""
    blk, dtype = case["block"], case["dtype"]
    nblk = scales.shape[2]
    old = scales.transpose(1, 2).reshape(-1, scales.shape[1])                 # [B * nblk, Hkv]
    slot = (seq * nblk + at // blk)
    amax = torch.zeros_like(old).index_reduce_(0, slot, new.abs().amax(dim=-1), "amax")
    scale = _need(amax, dtype)
    # A block that holds rows already keeps its scale unless it has to grow.
    b = torch.arange(lens.numel(), device="cuda")
    first = b * nblk + (lens // blk).clamp(max=nblk - 1)
    begun = (lens % blk != 0)[:, None]
    scale[first] = torch.where(begun, torch.maximum(scale[first], old[first]), scale[first])
    touched = torch.zeros(old.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, slot, True)
    scale = torch.where(touched[:, None], scale, old)
    # The rows that such a block held, to its new scale.
    rows = (lens // blk * blk)[:, None] + torch.arange(blk, device="cuda")
    held = rows < lens[:, None]
    rows = rows.clamp(max=codes.shape[1] - 1)
    raw = codes.view(torch.int8)
    was = raw[b[:, None], rows]
    ratio = (old[first] / scale[first])[:, None, :, None]
    moved = _codes(was.view(codes.dtype).float() * ratio, dtype).view(torch.int8)
    hb, hr = (b[:, None].expand_as(rows))[held], rows[held]
    raw[hb, hr] = moved[held]
    raw[seq, at] = _codes(new / scale[slot][..., None], dtype).view(torch.int8)
    scales.copy_(scale.view(scales.shape[0], nblk, -1).transpose(1, 2))


def _plain_append(s):
    case = s["case"]
    lens = s["lens"].long()
    cu = torch.tensor(s["cu"], device="cuda")
    row = torch.arange(s["cu"][-1], device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    at = lens[seq] + row - cu[seq]
    after = (lens + cu[1:] - cu[:-1]).to(torch.int32)
    for name in ("k", "v"):
        _plain_store(s[name], s[name + "_scales"], s["new_" + name].float().view(-1, case["heads_kv"], D),
                     seq, at, lens, case)
    rows = case["hi"] + case["block"] - 1
    return (after,) + tuple(_plain_rows(s[n], s[n + "_scales"], case["block"], s["starts"], rows, after)
                            for n in ("k", "v"))


def _plain_decode(s):
    case = s["case"]
    b, n, hq, hkv = case["batch"], case["capacity"], case["heads_q"], case["heads_kv"]
    g, c = hq // hkv, D ** -0.5 * math.log2(math.e)
    k = _values(s["k"], s["k_scales"], case["block"]).permute(0, 2, 3, 1).contiguous()
    x = torch.matmul(s["q"].float().view(b, hkv, g, D), k).mul_(c)
    j, lens = torch.arange(n, device="cuda"), s["lens"].long()[:, None]
    first = torch.where(s["full"][:, None], 0, (lens - case["window"]).clamp(min=0))
    x = x.masked_fill(~((j < lens) & (j >= first))[:, None, None], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    p = torch.exp2(x - top)
    total = p.sum(dim=-1, keepdim=True)
    p = p / total
    v = _values(s["v"], s["v_scales"], case["block"]).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(p, v).view(b, 1, hq, D).to(torch.bfloat16)
    lse = (top + torch.log2(total)).view(b, 1, hq)
    if not case["weights"]:
        return out, lse
    s["sums"].add_(p.sum(dim=2))
    return out, lse, s["sums"]


def _plain_evict(s):
    case = s["case"]
    n, budget, recent, blk = case["capacity"], case["budget"], case["recent"], case["block"]
    b, hkv = case["batch"], case["heads_kv"]
    lens, pos = s["lens"].long()[:, None, None], torch.arange(n, device="cuda")
    old = pos < lens - recent
    order = torch.sort(torch.where(old, s["sums"], -1.0), dim=-1, descending=True, stable=True).indices
    heavy = torch.zeros(b, hkv, n, dtype=torch.bool, device="cuda")
    heavy.scatter_(2, order[..., : budget - recent], True)
    keep = torch.where(lens > budget, (heavy & old) | ~old, True) & (pos < lens)
    to = torch.where(keep, torch.cumsum(keep, dim=-1) - 1, budget)
    src = torch.zeros(b, hkv, budget + 1, dtype=torch.long, device="cuda")
    src = src.scatter_(2, to, pos.expand(b, hkv, n))[..., :budget]
    after = lens.clamp(max=budget)
    live = torch.arange(budget, device="cuda") < after
    sums = torch.where(live, torch.gather(s["sums"], 2, src), 0.0)
    nblk = -(-budget // blk)
    ib, ih = torch.arange(b, device="cuda")[:, None, None], torch.arange(hkv, device="cuda")[:, None]

    def moved(codes, scales):
        x = codes.view(torch.uint8)[ib, src, ih].view(codes.dtype).float()
        x = x * torch.gather(scales, 2, src // blk)[..., None]
        x = torch.where(live[..., None], x, 0.0)
        x = torch.nn.functional.pad(x, (0, 0, 0, nblk * blk - budget)).view(b, hkv, nblk, blk, D)
        scale = _need(x.abs().amax(dim=(3, 4)), case["dtype"])[..., None, None]
        x = (_codes(x / scale, case["dtype"]).float() * scale).view(b, hkv, nblk * blk, D)
        return x[:, :, :budget].transpose(1, 2).to(torch.bfloat16)

    return (after.view(-1).to(torch.int32), sums, moved(s["k"], s["k_scales"]),
            moved(s["v"], s["v_scales"]))


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "append":
        return _plain_append(state)
    if op == "read":
        case = state["case"]
        return tuple(_plain_rows(state[n], state[n + "_scales"], case["block"], state["starts"],
                                 case["rows"], None) for n in ("k", "v"))
    if op == "decode":
        return _plain_decode(state)
    return _plain_weights(state) if op == "weights" else _plain_evict(state)


def _run_own(s):
    import switchattentionkernels_amd as swa

    case = s["case"]
    if case["op"] == "weights":
        return swa.switch_gqa_prefill_key_weights(s["q"], s["k"], s["lse"], s["full"], s["local"],
                                                  window_size=case["window"])
    cache = swa.SwitchKVCache(s["k"], s["v"], s["k_scales"], s["v_scales"], case["block"])
    if case["op"] == "append":
        after = swa.switch_kv_cache_append(cache, s["new_k"], s["new_v"], s["lens"],
                                           cu_seqlens=s["cu"] if case["packed"] else None)
        k, v = swa.switch_kv_cache_read(cache, s["starts"], case["hi"] + case["block"] - 1,
                                        cache_lens=after)
        return after, k, v
    if case["op"] == "read":
        return swa.switch_kv_cache_read(cache, s["starts"], case["rows"])
    if case["op"] == "decode":
        out, lse = swa.switch_gqa_decode_quantized_forward(
            s["q"], cache, s["lens"], s["full"], window_size=case["window"],
            key_weights=s["sums"] if case["weights"] else None)
        return (out, lse, s["sums"]) if case["weights"] else (out, lse)
    kept, after, sums = swa.switch_kv_cache_evict(cache, s["lens"], s["sums"], budget=case["budget"],
                                                  recent=case["recent"], capacity=case["budget"])
    k, v = swa.switch_kv_cache_read(kept, 0, case["budget"], cache_lens=after)
    return after, sums, k, v


# ---------------------------------------------------------------------------
# The work that a pass cannot do without
# ---------------------------------------------------------------------------
def _pairs(case):
    """Expected legal (query, key) pairs of one head."""
    n, w, p = case["seq"], min(case["window"], case["seq"]), case["p_full"]
    return case["batch"] * (p * n * (n + 1) / 2 + (1 - p) * (w * (w + 1) / 2 + (n - w) * w))


def work(case):
    op, hkv = case["op"], case["heads_kv"]
    if op == "weights":
        rows = case["batch"] * case["seq"]
        return {"bytes": rows * (case["heads_q"] * (2 * D + 4) + hkv * (2 * D + 4) + 4),
                "flops": 2 * D * case["heads_q"] * _pairs(case)}
    coded, plain = 2 * D + 8 / case["block"], 4 * D       # bytes of a row's K and V for one head
    if op == "append":
        rows, began = sum(_new_rows(case)), sum(x % case["block"] for x in _old_lens(case))
        out = case["batch"] * (case["hi"] + case["block"] - 1)
        return {"bytes": hkv * (rows * (plain + coded) + (rows + began) * coded + out * plain),
                "flops": hkv * 2 * D * (3 * rows + out)}
    if op == "read":
        rows = case["batch"] * case["rows"]
        return {"bytes": rows * hkv * (coded + plain), "flops": rows * hkv * 2 * D}
    if op == "decode":
        lens, full = _decode_lens(case), _decode_full(case)
        keys = sum(n if f else min(n, case["window"]) for n, f in zip(lens, full))
        hq = case["heads_q"]
        return {"bytes": keys * hkv * (coded + (8 if case["weights"] else 0)) +
                case["batch"] * hq * (4 * D + 4), "flops": 4 * D * hq * keys}
    lens = _evict_lens(case)
    kept = sum(min(n, case["budget"]) for n in lens)
    out = case["batch"] * case["budget"]
    return {"bytes": hkv * (sum(lens) * 4 + kept * 3 * coded + out * (plain + 4)),
            "flops": hkv * 2 * D * 3 * kept}


# ---------------------------------------------------------------------------
# The same in 64 bits, by other means
# ---------------------------------------------------------------------------
def _exact_scale(amax, dtype):
    """Search in the table of the largest magnitudes that powers of two hold."""
    e = np.arange(MIN_EXP, 128)
    return np.ldexp(1.0, e[np.searchsorted(QMAX[dtype] * np.ldexp(1.0, e), amax, side="left")])


def _exact_round(x, dtype):
    """To the nearest code, ties to the even one."""
    if dtype == "int8":
        return np.rint(x)
    step = np.ldexp(1.0, np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 1e-300))), -6).astype(int) - 3)
    return np.rint(x / step) * step


def _np(t):
    return t.float().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _exact_append(s, case):
    lens, cu, blk = _np(s["lens"]), s["cu"], case["block"]
    rows = case["hi"] + blk - 1
    outs = []
    for name in ("k", "v"):
        new = _np(s["new_" + name]).reshape(-1, case["heads_kv"], D)
        codes, scales = _np(s[name]), _np(s[name + "_scales"])
        out = np.zeros((case["batch"], rows, case["heads_kv"], D))
        for b in range(case["batch"]):
            fresh, begin = new[cu[b]:cu[b + 1]], int(s["starts"][b])
            held = int(lens[b]) - begin
            here = scales[b, :, begin // blk] if held else None      # the scale of the begun block
            old = codes[b, begin:begin + held] * (here[:, None] if held else 1.0)
            x = np.concatenate([old, fresh])
            for at in range(0, len(x), blk):
                part = x[at:at + blk]
                skip = held if at == 0 else 0
                scale = _exact_scale(np.abs(part[skip:]).max(axis=(0, 2)), case["dtype"])
                if skip:
                    scale = np.maximum(scale, here)
                out[b, at:at + len(part)] = _exact_round(part / scale[:, None], case["dtype"]) * scale[:, None]
        outs.append(out)
    return [None] + outs


def _exact_rows(codes, scales, blk, starts, rows):
    b = np.arange(codes.shape[0])[:, None]
    at = starts[:, None] + np.arange(rows)
    return codes[b, at] * np.swapaxes(scales, 1, 2)[b, at // blk][..., None]


def _exact_decode(s, case):
    b, hq, hkv, blk = case["batch"], case["heads_q"], case["heads_kv"], case["block"]
    g = hq // hkv
    out, lse = torch.empty(b, 1, hq, D, dtype=torch.float64), torch.empty(b, 1, hq, dtype=torch.float64)
    sums = s["sums"].double() if case["weights"] else None
    for i in range(b):
        n = int(s["lens"][i])
        lo = 0 if bool(s["full"][i]) else max(n - case["window"], 0)
        at = torch.arange(lo, n, device="cuda")
        k, v = (s[x][i, lo:n].to(torch.float32).double() * s[x + "_scales"][i].double().t()[at // blk][..., None]
                for x in ("k", "v"))
        q = s["q"][i, 0].double().view(hkv, g, D)
        x = torch.matmul(k.transpose(0, 1).contiguous(), q.transpose(1, 2).contiguous()) / math.sqrt(D)
        z = torch.logsumexp(x, dim=1, keepdim=True)                   # [hkv, keys, g] over the keys
        p = torch.exp(x - z)
        out[i, 0] = torch.matmul(p.transpose(1, 2).contiguous(), v.transpose(0, 1).contiguous()).view(hq, D).cpu()
        lse[i, 0] = (z / math.log(2.0)).reshape(hq).cpu()
        if sums is not None:
            sums[i, :, lo:n] += p.sum(dim=2)
    return (out, lse, sums) if case["weights"] else (out, lse)


def _exact_weights(s, case):
    b, n, hq, hkv = case["batch"], case["seq"], case["heads_q"], case["heads_kv"]
    local = torch.zeros(b * n, dtype=torch.bool, device="cuda").index_fill_(0, s["local"].long(), True).view(b, n)
    sums = torch.zeros(b, hkv, n, dtype=torch.float64, device="cuda")
    j = torch.arange(n, device="cuda")
    for i in range(b):
        for h in range(hq):
            kh = s["k"][i, :, h // (hq // hkv)].double().t().contiguous()
            for r in range(0, n, 4096):                               # blocks of queries
                rows = torch.arange(r, min(n, r + 4096), device="cuda")
                end = int(rows[-1]) + 1
                x = torch.matmul(s["q"][i, rows, h].double(), kh[:, :end]) / math.sqrt(D)
                x = torch.exp(x - s["lse"][i, rows, h].double()[:, None] * math.log(2.0))
                far = rows[:, None] - j[:end]
                x[(far < 0) | (local[i, rows][:, None] & (far >= case["window"]))] = 0.0
                sums[i, h // (hq // hkv), :end] += x.sum(dim=0)
    return sums


def _exact_evict(s, case):
    blk, budget, recent = case["block"], case["budget"], case["recent"]
    lens, sums = _np(s["lens"]), _np(s["sums"])
    ks, vs = _np(s["k_scales"]), _np(s["v_scales"])
    k, v = _np(s["k"]), _np(s["v"])
    shape = (case["batch"], budget, case["heads_kv"])
    ok, ov, ow = np.zeros(shape + (D,)), np.zeros(shape + (D,)), np.zeros((shape[0], shape[2], budget))
    for b in range(case["batch"]):
        for h in range(case["heads_kv"]):
            n = int(lens[b])
            at = np.arange(n)
            if n > budget:
                first = at[: n - recent]
                best = np.lexsort((first, -sums[b, h, : n - recent]))[: budget - recent]
                at = np.concatenate([np.sort(best), at[n - recent:]])
            ow[b, h, : len(at)] = sums[b, h, at]
            for out, codes, scales in ((ok, k, ks), (ov, v, vs)):
                x = codes[b, at, h] * scales[b, h, at // blk][:, None]
                for r in range(0, len(at), blk):
                    sc = _exact_scale(np.abs(x[r:r + blk]).max(), case["dtype"])
                    out[b, r:min(r + blk, len(at)), h] = _exact_round(x[r:r + blk] / sc, case["dtype"]) * sc
    return [None, ow, ok, ov]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "append":
        return _exact_append(s, case)
    if op == "read":
        return [_exact_rows(_np(s[n]), _np(s[n + "_scales"]), case["block"], _np(s["starts"]), case["rows"])
                for n in ("k", "v")]
    if op == "decode":
        return _exact_decode(s, case)
    return _exact_weights(s, case) if op == "weights" else _exact_evict(s, case)
