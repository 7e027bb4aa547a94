"""Cases for the operators of one decode step over a paged key/value cache.

The operators, in the order in which a step calls them:

- qk_norm_rope: RMS norm of every query and key head, a learned weight per
  channel, and the rotation by position, in one pass; with its gradient.
- paged_attention: attention of one new token per sequence over a paged
  cache, and its scored form, which also adds each slot's attention weight
  (summed over the query heads that share the key head) to running scores.
- cache_evict: keeps `budget` slots of each sequence and key head, the
  newest, the first and the highest scored ones, and moves the kept rows that
  lie past the budget into the places that became free.

`run` computes them in plain torch where `own` is false, and through
porch_b200.api where it is true. `exact` computes them in 64 bits.
"""

import math
import random

import numpy as np
import torch

own = False


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # One new token of one sequence: the projections' heads before attention; latency.
        dict(name="norm_rope_one_token", op="norm_rope", tokens=1, q_heads=8, kv_heads=2, head_dim=64, rot=64,
             interleaved=False, table=4096),
        # A short prompt with odd head counts, a head size that is no power of two, a partly rotated head.
        dict(name="norm_rope_odd", op="norm_rope", tokens=1021, q_heads=15, kv_heads=5, head_dim=80, rot=40,
             interleaved=True, table=2048),
        # A long prompt or a training batch, read in place from a fused projection.
        dict(name="norm_rope_long", op="norm_rope", tokens=16384, q_heads=32, kv_heads=8, head_dim=128, rot=128,
             interleaved=False, table=8192),
        # The gradient at an odd number of tokens and a partly rotated head.
        dict(name="norm_rope_grad_odd", op="norm_rope_grad", tokens=777, q_heads=12, kv_heads=4, head_dim=96, rot=48,
             interleaved=False, table=1024),
        # The gradient of a training batch.
        dict(name="norm_rope_grad_long", op="norm_rope_grad", tokens=8192, q_heads=32, kv_heads=8, head_dim=128,
             rot=128, interleaved=False, table=4096),
        # The first steps of a single chat: a handful of slots; latency.
        dict(name="attend_one_short", op="attend", seqs=1, longest=37, q_heads=8, kv_heads=2, head_dim=64, page=16,
             dtype="bf16"),
        # A serving batch whose sequences differ in length, an empty one among them.
        dict(name="attend_batch_ragged", op="attend", seqs=48, longest=8191, q_heads=32, kv_heads=8, head_dim=128,
             page=64, dtype="bf16"),
        # One sequence with a very long context: few rows, a long axis.
        dict(name="attend_one_long", op="attend", seqs=1, longest=262147, q_heads=32, kv_heads=8, head_dim=128,
             page=128, dtype="bf16"),
        # A cache in 32 bits without shared heads.
        dict(name="attend_f32_batch", op="attend", seqs=16, longest=2049, q_heads=16, kv_heads=16, head_dim=64,
             page=16, dtype="f32"),
        # Decoding while the scores for eviction are gathered.
        dict(name="attend_scored_batch", op="attend_scored", seqs=16, longest=8200, q_heads=32, kv_heads=8,
             head_dim=128, page=32, dtype="bf16"),
        # The steady state: a few tokens past the budget after a few steps.
        dict(name="evict_after_steps", op="evict", seqs=24, longest=1048, kv_heads=8, head_dim=128, page=16,
             dtype="bf16", budget=1024, recent=128, sinks=4, seen=True),
        # Once after long prompts: most of the cache goes.
        dict(name="evict_after_prompt", op="evict", seqs=4, longest=65533, kv_heads=8, head_dim=128, page=64,
             dtype="bf16", budget=4096, recent=1024, sinks=4, seen=False),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _shape(rng):
    """Head size, key heads and query heads."""
    while True:
        dim, kv = rng.choice([64, 80, 96, 128, 256]), rng.choice([1, 2, 4, 5, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 6, 8])
        if 3 * 1024 not in (heads * dim, (heads + kv) * dim, (heads + 2 * kv) * dim):
            return dim, kv, heads


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope_grad", "attend", "attend", "attend_scored", "evict"])
    dim, kv, heads = _shape(rng)
    if op in ("norm_rope", "norm_rope_grad"):
        most = (16384 if op == "norm_rope" else 8192) * 40 * 128 // ((heads + kv) * dim)
        rot = rng.choice([dim, dim, dim // 2, 32])
        return dict(op=op, tokens=_spread(rng, 1, most), q_heads=heads, kv_heads=kv, head_dim=dim, rot=rot,
                    interleaved=rng.random() < 0.3, table=rng.choice([1024, 4096, 8192]))
    dtype = rng.choice(["bf16", "bf16", "f32"])
    page = rng.choice([8, 16, 32, 64, 128, 256])
    slot = 2 * kv * dim * (2 if dtype == "bf16" else 4)  # bytes of one cached token
    seqs = _spread(rng, 1, 64)
    if op != "evict":
        most = max(2, min(262144, (1 << 29) // (slot * seqs)))
        return dict(op=op, seqs=seqs, longest=_spread(rng, 1, most), q_heads=heads, kv_heads=kv, head_dim=dim,
                    page=page, dtype=dtype)
    most = max(256, min(65536, (1 << 29) // (slot * seqs)))
    longest = _spread(rng, 256, most)
    budget = _spread(rng, 64, longest)
    return dict(op=op, seqs=seqs, longest=longest, kv_heads=kv, head_dim=dim, page=page, dtype=dtype, budget=budget,
                recent=_spread(rng, 1, budget // 2), sinks=rng.choice([0, 4, 16]), seen=rng.random() < 0.5)


def _lengths(case):
    """Slots in use by each sequence; a rule of the case alone. A batch of
    8 or more sequences has an empty one."""
    n, longest = case["seqs"], case["longest"]
    if case["op"] == "evict":
        return [longest - (7 * i) % max(1, longest // 64) for i in range(n)]
    lens = [longest] + [1 + int((longest - 1) * ((0.618034 * i) % 1.0)) for i in range(1, n)]
    return [0 if n >= 8 and i == n // 2 else v for i, v in enumerate(lens)]


def _width(case):
    return 2 if case["dtype"] == "bf16" else 4


def work(case):
    if case["op"] in ("norm_rope", "norm_rope_grad"):
        t, d = case["tokens"], case["head_dim"]
        values = t * (case["q_heads"] + case["kv_heads"]) * d
        small = 4 * (t + 2 * d + min(t, case["table"]) * case["rot"])
        if case["op"] == "norm_rope":
            return dict(bytes=8 * values + small, flops=7 * values)
        return dict(bytes=12 * values + small + 8 * d, flops=18 * values)
    lens, d, kv = _lengths(case), case["head_dim"], case["kv_heads"]
    if case["op"] != "evict":
        slots, g = sum(lens), case["q_heads"] // kv
        moved = 2 * slots * kv * d * _width(case) + 8 * case["seqs"] * case["q_heads"] * d
        if case["op"] == "attend_scored":
            moved += 4 * slots * kv + 4 * case["seqs"] * kv * case["longest"]
        return dict(bytes=moved, flops=4 * slots * kv * g * d)
    budget, total = case["budget"], 0.0
    for n in lens:
        kept = min(n, budget)
        total += 4 * n + (4 * min(n, budget) if case["seen"] else 0) + 8 * budget
        fresh = min(case["recent"], n - kept)  # the newest slots that lie past the budget
        young = n - min(budget, min(lens)) if case["seen"] else n  # slots that can be among the newest
        safe = min(n, min(case["recent"], young) + case["sinks"])
        free, take = n - safe, max(0, kept - safe)
        rows = fresh + (take / free if free else 0.0) * max(0, n - kept - fresh)
        total += rows * 4 * d * _width(case)
    return dict(bytes=total * kv, flops=sum(lens) * kv)


# ------------------------------------------------------------------ inputs --
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)


def _norm_rope_inputs(case, seed):
    g = _generator(seed)
    t, hq, hk, d, r = (case[k] for k in ("tokens", "q_heads", "kv_heads", "head_dim", "rot"))
    # The fused projection of a layer: queries, keys and values of a token side by side.
    qkv = torch.randn(t, hq + 2 * hk, d, generator=g, device="cuda")
    qkv *= torch.rand(hq + 2 * hk, 1, generator=g, device="cuda") * 2 + 0.5
    s = dict(case=case, qkv=qkv, q_weight=1 + 0.2 * torch.randn(d, generator=g, device="cuda"),
             k_weight=1 + 0.2 * torch.randn(d, generator=g, device="cuda"))
    angle = (torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None]
             * 10000.0 ** (-torch.arange(r // 2, device="cuda", dtype=torch.float64) * 2 / r))
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    first = int(torch.randint(0, case["table"], (1,), generator=g, device="cuda"))
    s["positions"] = ((torch.arange(t, device="cuda") + first) % case["table"]).float()
    if case["op"] == "norm_rope_grad":
        s["dq"] = torch.randn(t, hq, d, generator=g, device="cuda")
        s["dk"] = torch.randn(t, hk, d, generator=g, device="cuda")
    return s


def _cache_inputs(case, seed):
    g = _generator(seed)
    lens, page, kv, d = _lengths(case), case["page"], case["kv_heads"], case["head_dim"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device="cuda").cpu().numpy()
    table = np.zeros((len(lens), max(1, max(counts))), dtype=np.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    s = dict(case=case, lens=lens, table=table, pages=pages)
    s["k"] = torch.randn(pages, kv, page, d, generator=g, device="cuda").to(dtype)
    s["v"] = torch.randn(pages, kv, page, d, generator=g, device="cuda").to(dtype)
    if case["op"] != "evict":
        s["q"] = 2 * torch.randn(len(lens), case["q_heads"], d, generator=g, device="cuda")
        if case["op"] == "attend_scored":
            s["scores"] = torch.rand(len(lens), kv, max(1, case["longest"] - 1), generator=g, device="cuda")
        return s
    # Few slots gather most of the weight, and some none at all.
    rows = (len(lens), kv, case["longest"])
    s["scores"] = torch.exp(2 * torch.randn(rows, generator=g, device="cuda"))
    s["scores"] *= torch.rand(rows, generator=g, device="cuda") > 0.1
    newest = [3 * n for n in lens] if case["seen"] else [n - 1 for n in lens]
    s["newest"], s["places"] = newest, None
    if case["seen"]:  # what an earlier eviction kept: older tokens, in no order
        b = min(case["budget"], min(lens))
        old = torch.rand(len(lens), kv, b, generator=g, device="cuda").argsort(-1)
        s["places"] = old.float()
    return s


def prepare(case, seed):
    """What a program holds before the call. Of the framework (`own`) that is
    its tensors, its cache and the batch's page tables; the same values."""
    if case["op"] in ("norm_rope", "norm_rope_grad"):
        s = _norm_rope_inputs(case, seed)
        if own:
            from porch_b200 import api

            hq, hk = case["q_heads"], case["kv_heads"]
            mine = {k: api.tensor_from_device(v) for k, v in s.items() if k != "case"}
            heads = mine.pop("qkv")
            mine["q"] = api.materialize(heads[api.all, 0:hq, api.all])
            mine["k"] = api.materialize(heads[api.all, hq:hq + hk, api.all])
            s = dict(case=case, **mine)
        return s
    s = _cache_inputs(case, seed)
    if own:
        from porch_b200 import api

        cache = api.KVCache(s["pages"], case["page"], case["kv_heads"], case["head_dim"], dtype=case["dtype"])
        pools = _pools(cache, case)
        pools[0].copy_(s["k"])
        pools[1].copy_(s["v"])
        torch.cuda.synchronize()
        mine = dict(case=case, cache=cache, pools=pools,
                    batch=cache.batch(s["table"], s["lens"], newest=s.get("newest")))
        for name in ("q", "scores", "places"):
            mine[name] = api.tensor_from_device(s[name]) if s.get(name) is not None else None
        s = mine
    else:
        s["length"] = torch.tensor(s["lens"], device="cuda")
        s["table"] = torch.from_numpy(s["table"]).cuda().long()
        if "newest" in s:
            s["last"] = torch.tensor(s["newest"], device="cuda")
    return s


def _pools(cache, case):
    k, v = (torch.as_tensor(p, device="cuda") for p in cache.pools())
    return (k.view(torch.bfloat16), v.view(torch.bfloat16)) if case["dtype"] == "bf16" else (k, v)


# --------------------------------------------------------------- plain form --
def _turn(x, cos, sin, rot, interleaved):
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _heads(s):
    hq, hk = s["case"]["q_heads"], s["case"]["kv_heads"]
    return s["qkv"][:, :hq], s["qkv"][:, hq:hq + hk]


def _rows(s):
    at = s["positions"].long()
    return s["cos"][at][:, None], s["sin"][at][:, None]


def _norm_rope(x, weight, cos, sin, case):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    return _turn(x * r * weight, cos, sin, case["rot"], case["interleaved"])


def _norm_rope_grad(dy, x, weight, cos, sin, case):
    g = _turn(dy, cos, -sin, case["rot"], case["interleaved"])
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    normed = x * r
    gw = g * weight
    dx = r * (gw - normed * (gw * normed).mean(-1, keepdim=True))
    return dx, (g * normed).sum((0, 1))


def _gathered(s, pool):
    """[sequences, heads, slots, head_dim] in 32 bits, padded to whole pages of the longest."""
    x = pool[s["table"]].transpose(1, 2)  # [S, H, pages, page, D]
    return x.flatten(2, 3).float()


def _attend(s):
    case = s["case"]
    n, kv, d = case["seqs"], case["kv_heads"], case["head_dim"]
    k, v = _gathered(s, s["k"]), _gathered(s, s["v"])
    q = s["q"].view(n, kv, -1, d) * d ** -0.5
    logits = q @ k.transpose(-1, -2)  # [S, H, G, slots]
    seen = torch.arange(k.shape[2], device="cuda") < s["length"][:, None]
    logits = logits.masked_fill(~seen[:, None, None], float("-inf"))
    top = logits.amax(-1, keepdim=True).clamp_min(-3.0e38)
    p = torch.exp(logits - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    v = v.masked_fill(~seen[:, None, :, None], 0.0)
    return (p @ v).reshape(n, -1, d), p


def _evict(s):
    case = s["case"]
    budget, scores, page = case["budget"], s["scores"], case["page"]
    n, kv, c = scores.shape
    slot = torch.arange(c, device="cuda").expand(n, kv, c)
    length, last = s["length"][:, None, None], s["last"][:, None, None]
    place = last - (length - 1 - slot)
    if s["places"] is not None:
        b = s["places"].shape[-1]
        place = torch.cat((torch.where(s["places"] >= 0, s["places"].long(), place[..., :b]), place[..., b:]), -1)
    safe = (place > last - case["recent"]) | (place < case["sinks"])
    key = torch.where(scores.isnan(), float("-inf"), scores).clamp_max(3.0e38)
    key = torch.where(safe, float("inf"), key).masked_fill(slot >= length, float("-inf"))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.zeros(n, kv, c, dtype=torch.bool, device="cuda").scatter_(-1, order, True) & (slot < length)
    hole = ~kept & (slot < budget) & (slot < length)
    late = kept & (slot >= budget)
    # The j-th kept slot past the budget fills the j-th hole.
    at = torch.zeros(n, kv, c + 1, dtype=torch.long, device="cuda")
    at.scatter_(-1, torch.where(late, late.cumsum(-1) - 1, c), slot)
    source = torch.where(hole, at.gather(-1, (hole.cumsum(-1) - 1).clamp_min(0)), slot)[..., :budget]
    live = torch.arange(source.shape[-1], device="cuda") < torch.minimum(length, torch.tensor(budget, device="cuda"))
    empty = budget - source.shape[-1]
    out = torch.where(live, scores.gather(-1, source), 0.0)
    where = torch.where(live, place.gather(-1, source), -1).float()
    # Rows move inside the pools: [page, head, place in the page].
    i, h, j = torch.nonzero(hole[..., :budget], as_tuple=True)
    head = torch.arange(kv, device="cuda")

    def row(x):
        return (s["table"][i, x // page] * kv + head[h]) * page + x % page

    to, frm = row(j), row(source[i, h, j])
    for_k, for_v = (p.view(-1, p.shape[-1]) for p in (s["k"], s["v"]))
    for_k[to] = for_k[frm]
    for_v[to] = for_v[frm]
    pad = torch.nn.functional.pad
    return pad(out, (0, empty)), pad(where, (0, empty), value=-1.0), s["k"], s["v"]


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        return _run_own(s, case, op)
    if op == "norm_rope":
        q, k = _heads(s)
        cos, sin = _rows(s)
        return _norm_rope(q, s["q_weight"], cos, sin, case), _norm_rope(k, s["k_weight"], cos, sin, case)
    if op == "norm_rope_grad":
        q, k = _heads(s)
        cos, sin = _rows(s)
        dq, dwq = _norm_rope_grad(s["dq"], q, s["q_weight"], cos, sin, case)
        dk, dwk = _norm_rope_grad(s["dk"], k, s["k_weight"], cos, sin, case)
        return dq, dk, dwq, dwk
    if op == "attend":
        return _attend(s)[0]
    if op == "attend_scored":
        out, p = _attend(s)
        p = p.sum(2)[..., :case["longest"]]
        seen = torch.arange(case["longest"], device="cuda") < s["length"][:, None, None]
        before = torch.nn.functional.pad(s["scores"], (0, case["longest"] - s["scores"].shape[-1]))
        return out, torch.where(seen, before[..., :case["longest"]] + p, 0.0)
    return _evict(s)


def _run_own(s, case, op):
    from porch_b200 import api

    if op == "norm_rope":
        out = api.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"],
                               eps=1e-6, interleaved=case["interleaved"])
    elif op == "norm_rope_grad":
        out = api.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"],
                                        s["sin"], s["positions"], eps=1e-6, interleaved=case["interleaved"])
    elif op == "attend":
        out = (api.paged_attention(s["q"], s["batch"]),)
    elif op == "attend_scored":
        out = api.paged_attention_scored(s["q"], s["batch"], s["scores"])
    else:
        out = api.cache_evict(s["batch"], s["scores"], s["places"], budget=case["budget"], recent=case["recent"],
                              sinks=case["sinks"])
    seen = tuple(torch.as_tensor(t, device="cuda") for t in out)
    if op == "evict":
        return seen + s["pools"]
    return seen[0] if op == "attend" else seen


# ------------------------------------------------------------------ 64 bits --
def exact(case, seed):
    if case["op"] in ("norm_rope", "norm_rope_grad"):
        return _exact_norm_rope(case, seed)
    if case["op"] == "evict":
        return _exact_evict(case, seed)
    return _exact_attend(case, seed)


def _exact_norm_rope(case, seed):
    s = _norm_rope_inputs(case, seed)
    rot, at = case["rot"], s["positions"].long()
    phase = torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None]

    def forward(x, w):
        y = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w
        head = y[..., :rot].unflatten(-1, (rot // 2, 2) if case["interleaved"] else (2, rot // 2))
        pair = 1 if case["interleaved"] else 0
        a, b = head.unbind(-1 if pair else -2)
        z = torch.complex(a, b) * phase
        return torch.cat((torch.stack((z.real, z.imag), -1 if pair else -2).flatten(-2), y[..., rot:]), -1)

    hq, hk = case["q_heads"], case["kv_heads"]
    x = [s["qkv"][:, :hq].double(), s["qkv"][:, hq:hq + hk].double()]
    w = [s["q_weight"].double(), s["k_weight"].double()]
    if case["op"] == "norm_rope":
        return forward(x[0], w[0]), forward(x[1], w[1])
    grads = []
    for xi, wi, dy in zip(x, w, (s["dq"], s["dk"])):
        xi.requires_grad_(True), wi.requires_grad_(True)
        grads.append(torch.autograd.grad(forward(xi, wi), (xi, wi), dy.double()))
    return grads[0][0], grads[1][0], grads[0][1], grads[1][1]


def _exact_attend(case, seed):
    s = _cache_inputs(case, seed)
    kv, d = case["kv_heads"], case["head_dim"]
    out = torch.zeros(case["seqs"], case["q_heads"], d, dtype=torch.float64, device="cuda")
    total = torch.zeros(case["seqs"], kv, case["longest"], dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["lens"]):
        if n == 0:
            continue
        at = torch.from_numpy(s["table"][i, :-(-n // case["page"])]).cuda().long()
        for h in range(kv):
            k, v = (p[at, h].reshape(-1, d)[:n].double() for p in (s["k"], s["v"]))
            q = s["q"][i].unflatten(0, (kv, -1))[h].double()
            p = torch.softmax(q @ k.T / math.sqrt(d), -1)
            out[i].unflatten(0, (kv, -1))[h] = p @ v
            total[i, h, :n] = p.sum(0)
    if case["op"] == "attend":
        return out
    for i, n in enumerate(s["lens"]):
        m = min(n, s["scores"].shape[-1])
        total[i, :, :m] += s["scores"][i, :, :m].double()
    return out, total


def _exact_evict(case, seed):
    s = _cache_inputs(case, seed)
    scores, budget = s["scores"].cpu().numpy(), case["budget"]
    places = None if s["places"] is None else s["places"].cpu().numpy()
    kv = case["kv_heads"]
    if len(s["lens"]) * kv * case["longest"] > 1 << 23:
        return None
    kept_scores = np.zeros((len(s["lens"]), kv, budget))
    kept_places = np.full((len(s["lens"]), kv, budget), -1.0)
    for i, n in enumerate(s["lens"]):
        for h in range(kv):
            place = np.arange(n) + (s["newest"][i] - (n - 1))
            if places is not None:
                b = min(n, places.shape[-1])
                place[:b] = places[i, h, :b]
            safe = (place > s["newest"][i] - case["recent"]) | (place < case["sinks"])
            order = np.lexsort((np.arange(n), -scores[i, h, :n], ~safe))[:budget]
            kept = np.zeros(n, dtype=bool)
            kept[order] = True
            source = np.arange(min(n, budget))
            source[~kept[:budget]] = np.flatnonzero(kept[budget:]) + budget
            kept_scores[i, h, :len(source)] = scores[i, h, source]
            kept_places[i, h, :len(source)] = place[source]
    return kept_scores, kept_places, None, None
