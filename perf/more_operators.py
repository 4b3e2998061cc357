"""Performance cases of what stands between a layer's projections and its decode
attention, and of that attention over a shared prefix.

* ``rotate``: queries and keys of a prompt, as the slices of one fused projection
  that they are, normalised per head (RMS, with a learnt weight, or not at all) and
  rotated by their positions in the same pass (``switch_qk_rotary_forward``).
  Positions have one axis, or three (time, height and width of image and video
  tokens) that share out the frequencies.
* ``train``: the same in a training step, forward and gradients of queries, keys
  and weights (``switch_qk_rotary``).
* ``append``: new tokens of a serving batch, one each or a ragged chunk: queries
  rotated, keys rotated into the bf16 cache behind each sequence's valid rows, values
  copied there (``switch_qk_rotary_append``).
* ``shared``: one routed decode step of a batch whose sequences continue shared
  prefixes (a system prompt, a document): every prefix is kept once, each sequence
  has a cache of its own rows behind it (``switch_gqa_decode_shared_forward``).

head_dim is 128 throughout and rows are bf16.  Sizes come from
``switchattentionkernels_amd/workloads.py`` and ``bench.py`` or are generic.
"""

from __future__ import annotations

import math
import random

import torch

own = False

D = 128
EPS = 1e-6


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _rows(op, batch, seq, heads_q, heads_kv, norm, rotary, axes, pairs, base, far, **more):
    """``norm``: type of the norms' weights ("fp32", "bf16") or "none"; ``rotary``:
    dims that are rotated; ``pairs``: neighbouring dims form a pair (else a dim and the
    one half of ``rotary`` further on); ``far``: largest position."""
    return {"op": op, "batch": batch, "seq": seq, "heads_q": heads_q, "heads_kv": heads_kv,
            "norm": norm, "rotary": rotary, "axes": axes, "pairs": pairs, "base": base,
            "far": far, **more}


def _shared(batch, heads_q, heads_kv, prefixes, prefix, capacity, window, p_full):
    """``prefixes`` prefixes of up to ``prefix`` rows (with more than one, lengths differ
    and some sequences have none); own rows up to ``capacity``."""
    return {"op": "shared", "batch": batch, "heads_q": heads_q, "heads_kv": heads_kv,
            "prefixes": prefixes, "prefix": prefix, "capacity": capacity, "window": window,
            "p_full": p_full}


def listed():
    return [
        # A short prompt on a small layer: the smallest rotation, latency only.
        dict(_rows("rotate", 1, 1024, 8, 2, "fp32", 128, 1, False, 1e4, 1023), name="rotate_s1024"),
        # Image tokens: three axes, a ragged length, five query heads per KV head.
        dict(_rows("rotate", 2, 2999, 40, 8, "bf16", 128, 3, False, 1e6, 4095),
             name="rotate_axes_b2_s2999"),
        # A long prompt, the benchmark's shape, at far positions.
        dict(_rows("rotate", 1, 16384, 32, 8, "fp32", 128, 1, False, 1e6, 131071), name="rotate_s16k"),
        # Training on short sequences with a small layer: half of the dims rotated, in pairs.
        dict(_rows("train", 1, 1024, 8, 2, "fp32", 64, 1, True, 1e4, 1023), name="train_s1024"),
        # Training at an ordinary length on a layer without norms, three axes.
        dict(_rows("train", 2, 4096, 32, 8, "none", 128, 3, False, 1e6, 4095), name="train_axes_b2_s4096"),
        # Long-context training, the benchmark's shape.
        dict(_rows("train", 1, 16384, 32, 8, "fp32", 128, 1, False, 1e6, 16383), name="train_s16k"),
        # One decode step's new token of a serving batch: latency only.
        dict(_rows("append", 64, 1, 32, 8, "bf16", 128, 1, False, 1e6, 32767, capacity=512),
             name="append_token_b64"),
        # A ragged chunk of eight prompts.
        dict(_rows("append", 8, 517, 64, 8, "fp32", 128, 1, False, 1e6, 8191, capacity=2048),
             name="append_chunk_b8"),
        # A few users of one short system prompt: the smallest step, latency only.
        dict(_shared(4, 8, 2, 1, 1024, 256, 256, 0.5), name="shared_b4_p1024"),
        # A ragged batch over three documents, five query heads per KV head, half of
        # the tokens routed full, some sequences without a document.
        dict(_shared(40, 40, 8, 3, 2999, 777, 512, 0.5), name="shared_docs_b40_p2999"),
        # A serving batch behind one long system prompt, routed as the benchmark is.
        dict(_shared(64, 32, 8, 1, 8192, 1024, 1024, 0.25), name="shared_b64_p8k"),
        # Many samples of one long document, all routed full, eight query heads per KV
        # head: the largest.
        dict(_shared(64, 64, 8, 1, 32768, 1024, 4096, 1.0), name="shared_b64_p32k"),
    ]


_HEADS = [(8, 2), (32, 8), (40, 8), (64, 8), (4, 1)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    """One more case of the listed ones' ranges."""
    op = rng.choice(["rotate", "train", "append", "shared", "shared"])
    heads_q, heads_kv = rng.choice(_HEADS)
    if op == "shared":
        batch = _log_int(rng, 1, 64)
        prefixes = rng.choice([1, 1, 2, 3])
        return _shared(batch, heads_q, heads_kv, prefixes, _log_int(rng, 256, 32768 // prefixes),
                       _log_int(rng, 64, 1024), _log_int(rng, 256, 4096),
                       rng.choice([0.0, 0.25, 0.5, 1.0]))
    style = (rng.choice(["none", "bf16", "fp32", "fp32"]), rng.choice([64, 96, 128, 128]),
             rng.choice([1, 1, 3]), rng.random() < 0.3, rng.choice([1e4, 5e5, 1e6]))
    if op == "append":
        batch = _log_int(rng, 1, 64)
        seq = rng.choice([1, _log_int(rng, 1, max(1, 4096 // batch))])
        return _rows(op, batch, seq, heads_q, heads_kv, *style, _log_int(rng, 8192, 131072),
                     capacity=seq + _log_int(rng, 1, max(1, 16384 // batch)))
    batch = rng.choice([1, 1, 2, 4])
    seq = _log_int(rng, 128, (16384 if heads_q <= 32 else 8192) // batch)
    return _rows(op, batch, seq, heads_q, heads_kv, *style, _log_int(rng, seq, 131072))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _spread(lo, hi, n):
    """n lengths from lo to hi in equal steps (the longest alone for n = 1)."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _old_lens(case):
    return _spread(0, case["capacity"] - case["seq"], case["batch"])


def _counts(case):
    return _spread(max(1, case["seq"] // 4), case["seq"], case["batch"])[::-1]


def _prefix_lens(case):
    return _spread(max(1, case["prefix"] // 4), case["prefix"], case["prefixes"])


def _prefix_ids(case):
    """Every prefix in turn; with more than one, each eighth sequence has none (-1)."""
    n = case["prefixes"]
    return [-1 if n > 1 and i % 8 == 7 else i % n for i in range(case["batch"])]


def _own_lens(case):
    return _spread(max(1, case["capacity"] // 4), case["capacity"], case["batch"])


def _full(case):
    p = case["p_full"]
    return [math.floor((i + 1) * p) > math.floor(i * p) if p < 1 else True for i in range(case["batch"])]


def _tails(case):
    """Rows of its prefix that each sequence attends."""
    lens = _prefix_lens(case)
    out = []
    for i, own_rows, full in zip(_prefix_ids(case), _own_lens(case), _full(case)):
        n = lens[i] if i >= 0 else 0
        out.append(n if full else min(n, max(0, case["window"] - own_rows)))
    return out


def _sections(case):
    """Frequencies of each axis: all, or a quarter for time and the rest in halves."""
    n = case["rotary"] // 2
    return [n] if case["axes"] == 1 else [n // 4, (n - n // 4) // 2, n - n // 4 - (n - n // 4) // 2]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(gen, *shape):
    """bf16, tokens of different magnitude (a factor of about two either way)."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    size = torch.exp(0.35 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))
    return (x * size).to(torch.bfloat16)


def _positions(case, order):
    """int32 [axes, B, S]: consecutive tokens up to ``far``; with three axes the tokens of
    frames of 24 x 32 patches."""
    b, n = case["batch"], case["seq"]
    first = [order.randint(0, max(0, case["far"] + 1 - n)) for _ in range(b)]
    first[-1] = max(0, case["far"] + 1 - n)
    at = torch.arange(n, device="cuda")
    start = torch.tensor(first, device="cuda")[:, None]
    if case["axes"] == 1:
        return (start + at)[None].to(torch.int32)
    frame, y, x = at // 768, at // 32 % 24, at % 32
    return torch.stack([start + frame, start + y, start + x]).to(torch.int32)


def prepare(case, seed):
    gen, order = _gen(seed), random.Random(int(seed))
    b, hq, hkv = case["batch"], case["heads_q"], case["heads_kv"]
    s = {"case": dict(case)}
    perm = list(range(b))
    order.shuffle(perm)
    pick = lambda values: [values[i] for i in perm]  # noqa: E731
    if case["op"] == "shared":
        for name in ("k", "v"):
            s[name + "_prefix"] = _normal(gen, case["prefixes"], case["prefix"], hkv, D)
            s[name + "_cache"] = _normal(gen, b, case["capacity"], hkv, D)
        s["q"] = torch.randn(b, 1, hq, D, generator=gen, device="cuda").to(torch.bfloat16)
        s["prefix_lens"], s["prefix_ids"] = _int32(_prefix_lens(case)), _int32(pick(_prefix_ids(case)))
        s["lens"] = _int32(pick(_own_lens(case)))
        s["full"] = torch.tensor(pick(_full(case)), device="cuda")
        return s
    n, r = case["seq"], case["rotary"]
    qkv = _normal(gen, b, n, hq + 2 * hkv, D)
    s["q"], s["k"], s["v"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], qkv[:, :, hq + hkv:]
    s["positions"] = _positions(case, order)
    s["inv_freq"] = case["base"] ** (torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / -r)
    s["axis"] = torch.repeat_interleave(torch.arange(case["axes"], device="cuda"),
                                        torch.tensor(_sections(case), device="cuda"))
    s["q_weight"] = s["k_weight"] = None
    if case["norm"] != "none":
        for name in ("q_weight", "k_weight"):
            w = 1.0 + 0.2 * torch.randn(D, generator=gen, device="cuda")
            s[name] = w.to(torch.bfloat16) if case["norm"] == "bf16" else w
    if case["op"] == "train":
        s["q"], s["k"] = s["q"].contiguous(), s["k"].contiguous()
        s["leaves"] = [s[x].requires_grad_() for x in ("q", "k", "q_weight", "k_weight") if s[x] is not None]
        s["grads"] = [_normal(gen, b, n, h, D) for h in (hq, hkv)]
    if case["op"] == "append":
        s["lens"], s["counts"] = _int32(pick(_old_lens(case))), _int32(pick(_counts(case)))
        s["k_cache"], s["v_cache"] = (_normal(gen, b, case["capacity"], hkv, D) for _ in range(2))
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_rows(s, x, weight):
    """fp32 of the rows x [B, S, H, D], normalised and rotated."""
    case = s["case"]
    r = case["rotary"]
    at = s["positions"][s["axis"]].permute(1, 2, 0).double()               # [B, S, R / 2]
    angle = (at * s["inv_freq"])[:, :, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight.float()
    if case["pairs"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _plain_rotate(s):
    return tuple(_plain_rows(s, s[x], s[x + "_weight"]).to(torch.bfloat16) for x in ("q", "k"))


def _plain_train(s):
    outs = _plain_rotate(s)
    return outs + torch.autograd.grad(outs, s["leaves"], s["grads"])


def _plain_append(s):
    q, k = _plain_rotate(s)
    capacity = s["case"]["capacity"]
    t = torch.arange(s["case"]["seq"], device="cuda")
    at = s["lens"].long()[:, None] + t
    live = (t < s["counts"].long()[:, None]) & (at < capacity)
    seq = torch.arange(s["case"]["batch"], device="cuda")[:, None].expand_as(at)
    s["k_cache"][seq[live], at[live]] = k[live]
    s["v_cache"][seq[live], at[live]] = s["v"][live]
    return q, (s["lens"] + s["counts"]).clamp(max=capacity), s["k_cache"], s["v_cache"]


def _plain_shared(s):
    case = s["case"]
    b, hq, hkv = case["batch"], case["heads_q"], case["heads_kv"]
    ids, lens = s["prefix_ids"].long(), s["lens"].long()[:, None]
    n, m = case["prefix"], case["capacity"]
    before = torch.where(ids >= 0, s["prefix_lens"].long()[ids], 0)[:, None]   # of its prefix
    # Logical position of every stored row, or -1.
    i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    at = torch.cat([torch.where(i < before, i, -1), torch.where(j < lens, before + j, -1)], dim=1)
    first = torch.where(s["full"][:, None], 0, (before + lens - case["window"]).clamp(min=0))
    hide = (at < first)[:, None, None]

    def rows(name, *order):
        x = torch.cat([s[name + "_prefix"][ids], s[name + "_cache"]], dim=1)
        return x.permute(0, *order).float().contiguous()

    x = torch.matmul(s["q"].float().view(b, hkv, hq // hkv, D), rows("k", 2, 3, 1))
    x = x.mul_(D ** -0.5 * math.log2(math.e)).masked_fill_(hide, -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    p = torch.exp2(x - top)
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p / total, rows("v", 2, 1, 3)).view(b, 1, hq, D).to(torch.bfloat16)
    return out, (top + torch.log2(total)).view(b, 1, hq)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "rotate":
        return _plain_rotate(state)
    if op == "train":
        return _plain_train(state)
    return _plain_append(state) if op == "append" else _plain_shared(state)


def _run_own(s):
    import switchattentionkernels_amd as swa

    case = s["case"]
    if case["op"] == "shared":
        return swa.switch_gqa_decode_shared_forward(
            s["q"], s["k_prefix"], s["v_prefix"], s["prefix_lens"], s["prefix_ids"], s["k_cache"],
            s["v_cache"], s["lens"], s["full"], window_size=case["window"])
    how = {"sections": _sections(case), "interleaved": case["pairs"], "q_weight": s["q_weight"],
           "k_weight": s["k_weight"], "eps": EPS}
    if case["op"] == "rotate":
        return swa.switch_qk_rotary_forward(s["q"], s["k"], s["positions"], s["inv_freq"], **how)
    if case["op"] == "train":
        outs = swa.switch_qk_rotary(s["q"], s["k"], s["positions"], s["inv_freq"], **how)
        return outs + torch.autograd.grad(outs, s["leaves"], s["grads"])
    q, lens = swa.switch_qk_rotary_append(
        s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["lens"], s["positions"], s["inv_freq"],
        row_counts=s["counts"], **how)
    return q, lens, s["k_cache"], s["v_cache"]


# ---------------------------------------------------------------------------
# The work that a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    b, hq, hkv = case["batch"], case["heads_q"], case["heads_kv"]
    if case["op"] == "shared":
        tails, ids, own_lens = _tails(case), _prefix_ids(case), _own_lens(case)
        mine = [n if f else min(n, case["window"]) for n, f in zip(own_lens, _full(case))]
        once = sum(max([t for t, i in zip(tails, ids) if i == p] + [0]) for p in range(case["prefixes"]))
        return {"bytes": (once + sum(mine)) * hkv * 4 * D + b * hq * (4 * D + 4),
                "flops": 4 * D * hq * (sum(tails) + sum(mine))}
    tokens = b * case["seq"]
    if case["op"] == "append":
        rows = sum(_counts(case))
        return {"bytes": 4 * D * (tokens * hq + rows * 2 * hkv) + 4 * tokens * case["axes"],
                "flops": D * 9 * (tokens * hq + rows * hkv)}
    passes = {"rotate": 2, "train": 5 if case["norm"] != "none" else 4}[case["op"]]
    return {"bytes": tokens * ((hq + hkv) * 2 * D * passes + 4 * case["axes"]),
            "flops": D * tokens * (hq + hkv) * (9 if passes == 2 else 24)}


# ---------------------------------------------------------------------------
# The same in 64 bits, by other means
# ---------------------------------------------------------------------------
def _unit(s):
    """exp(i angle), complex [B, S, 1, R / 2], axis after axis."""
    parts, done = [], 0
    for axis, n in enumerate(_sections(s["case"])):
        a = s["positions"][axis].double()[..., None] * s["inv_freq"][done:done + n]
        parts.append(torch.polar(torch.ones_like(a), a))
        done += n
    return torch.cat(parts, dim=-1)[:, :, None]


def _turn(x, unit, case):
    """Rows x [B, S, H, D] times the unit numbers, each pair of dims as one complex number."""
    r = case["rotary"]
    y = x.clone()
    if case["pairs"]:
        z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * unit
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * unit
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y


def _exact_rows(s, name):
    x, w = s[name].detach().double(), s[name + "_weight"]
    if w is not None:
        x = x / torch.sqrt(x.square().sum(dim=-1, keepdim=True) / D + EPS) * w.detach().double()
    return _turn(x, _unit(s), s["case"])


def _exact_grads(s):
    dx, dw = [], []
    for name, dy in zip(("q", "k"), s["grads"]):
        g = _turn(dy.double(), _unit(s).conj(), s["case"])
        w = s[name + "_weight"]
        if w is None:
            dx.append(g)
            continue
        x = s[name].detach().double()
        size = torch.sqrt(x.square().sum(dim=-1, keepdim=True) / D + EPS)
        dw.append((g * x / size).sum(dim=(0, 1, 2)))
        g = g * w.detach().double()
        dx.append(g / size - x * (g * x).sum(dim=-1, keepdim=True) / (D * size ** 3))
    return dx + dw


def _exact_append(s):
    caches = [s[x].double() for x in ("k_cache", "v_cache")]
    for b, (n, count) in enumerate(zip(s["lens"].tolist(), s["counts"].tolist())):
        count = min(count, s["case"]["capacity"] - n)
        for cache, rows in zip(caches, (s["k_exact"], s["v"].double())):
            cache[b, n:n + count] = rows[b, :count]
    return caches


def _exact_shared(s, case):
    b, hq, hkv = case["batch"], case["heads_q"], case["heads_kv"]
    out = torch.empty(b, 1, hq, D, dtype=torch.float64)
    lse = torch.empty(b, 1, hq, dtype=torch.float64)
    lens, ids, before = s["lens"].tolist(), s["prefix_ids"].tolist(), s["prefix_lens"].tolist()
    for i in range(b):
        k, v = (torch.cat([s[x + "_prefix"][ids[i], :before[ids[i]]] if ids[i] >= 0 else
                           s[x + "_prefix"][0, :0], s[x + "_cache"][i, :lens[i]]]) for x in ("k", "v"))
        if not bool(s["full"][i]):
            k, v = k[-case["window"]:], v[-case["window"]:]
        q = s["q"][i, 0].double().view(hkv, hq // hkv, D)
        x = torch.matmul(k.double().transpose(0, 1).contiguous(), q.transpose(1, 2).contiguous()) / math.sqrt(D)
        z = torch.logsumexp(x, dim=1, keepdim=True)
        p = torch.exp(x - z).transpose(1, 2).contiguous()
        out[i, 0] = torch.matmul(p, v.double().transpose(0, 1).contiguous()).view(hq, D).cpu()
        lse[i, 0] = (z / math.log(2.0)).reshape(hq).cpu()
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "shared":
        return _exact_shared(s, case)
    q, k = _exact_rows(s, "q"), _exact_rows(s, "k")
    if case["op"] == "rotate":
        return q, k
    if case["op"] == "train":
        return [q, k] + _exact_grads(s)
    s["k_exact"] = k
    return [q, None] + _exact_append(s)
