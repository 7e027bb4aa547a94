"""Cases for operators of serving and of training on what a model says: a
key/value cache in 8 bits, attention of sequences that share a prefix, and the
log probabilities of given tokens.

- write_read: a step's new keys and values go into an int8 paged cache, a scale
  for each row (one token, one key head), and the sequences' slots are read back.
  A row's scale is its largest size / 127, its codes are the values / scale
  rounded to nearest, ties to even.
- attend: attention of one new token per sequence over such a cache.
- shared: the same for sequences whose first slots lie on the same pages (a
  system prompt, one question's many answers), which are worked through once for
  all of them.
- logprobs: for each row of logits the log probability of a given token (0 where
  it is -1, a padded row), the entropy, the row's largest logit beside the sum of
  exponentials relative to it, and the `top` likeliest tokens with their log
  probabilities (equal ones: the lower token first).
- logprobs_grad: the logits' gradient from those of the log probabilities and
  entropies.

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
        # A few short prompts written to the cache and read back; latency.
        dict(name="write_read_short", op="write_read", seqs=3, longest=29, fresh=29, kv_heads=2, head_dim=64, page=16),
        # A chunk of long prompts goes in, and the whole context is read back for a prefill that follows.
        dict(name="write_read_long", op="write_read", seqs=6, longest=16381, fresh=4096, kv_heads=8, head_dim=128,
             page=64),
        # The first steps of a single chat; latency.
        dict(name="attend_int8_short", op="attend", seqs=1, longest=45, q_heads=8, kv_heads=2, head_dim=64, page=16,
             dtype="int8"),
        # A serving batch whose sequences differ in length, an empty one among them.
        dict(name="attend_int8_ragged", op="attend", seqs=48, longest=8191, q_heads=32, kv_heads=8, head_dim=128,
             page=64, dtype="int8"),
        # One sequence with a very long context: few rows, a long axis.
        dict(name="attend_int8_one_long", op="attend", seqs=1, longest=262147, q_heads=32, kv_heads=8, head_dim=128,
             page=128, dtype="int8"),
        # A few answers to each of two questions, an odd head size.
        dict(name="shared_few", op="shared", groups=2, seqs=3, prefix=2016, longest=133, q_heads=15, kv_heads=5,
             head_dim=80, page=16, dtype="bf16"),
        # A serving batch behind one long system prompt.
        dict(name="shared_many", op="shared", groups=1, seqs=64, prefix=16384, longest=777, q_heads=32, kv_heads=8,
             head_dim=128, page=64, dtype="bf16"),
        # One sampled token with its alternatives; latency.
        dict(name="logprobs_one_row", op="logprobs", rows=1, vocab=32000, top=5),
        # A decoding batch that reports alternatives.
        dict(name="logprobs_step", op="logprobs", rows=64, vocab=131072, top=20),
        # The targets of a training batch, a vocabulary of odd size.
        dict(name="logprobs_long", op="logprobs", rows=4093, vocab=50257, top=0),
        # The gradient for a short batch, and for a training batch with an entropy bonus.
        dict(name="logprobs_grad_odd", op="logprobs_grad", rows=37, vocab=50257, entropy=False),
        dict(name="logprobs_grad_long", op="logprobs_grad", rows=4096, vocab=65536, entropy=True),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["write_read", "attend", "attend", "shared", "shared", "logprobs", "logprobs_grad"])
    if op in ("logprobs", "logprobs_grad"):
        vocab = _spread(rng, 500, 262144)
        rows = _spread(rng, 1, min(8192, (1 << 27) // vocab))
        if op == "logprobs":
            return dict(op=op, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]))
        return dict(op=op, rows=rows, vocab=vocab, entropy=rng.random() < 0.5)
    dim, kv = rng.choice([64, 80, 96, 128, 256]), rng.choice([1, 2, 4, 5, 8])
    page = rng.choice([8, 16, 32, 64, 128, 256])
    if op == "write_read":
        seqs = _spread(rng, 1, 64)
        longest = _spread(rng, 1, max(2, min(32768, (1 << 26) // (kv * dim * seqs))))
        return dict(op=op, seqs=seqs, longest=longest, fresh=_spread(rng, 1, longest), kv_heads=kv, head_dim=dim,
                    page=page)
    heads = kv * rng.choice([1, 2, 3, 4, 6, 8])
    if op == "attend":
        seqs = _spread(rng, 1, 64)
        most = max(2, min(262144, (1 << 28) // (kv * dim * seqs)))
        return dict(op=op, seqs=seqs, longest=_spread(rng, 1, most), q_heads=heads, kv_heads=kv, head_dim=dim,
                    page=page, dtype="int8")
    groups, seqs = rng.choice([1, 1, 2, 3]), _spread(rng, 2, 64)
    most = max(page, min(32768, (1 << 31) // (groups * seqs * heads * dim)))
    prefix = max(page, _spread(rng, page, most) // page * page)
    longest = _spread(rng, 1, max(2, min(2048, (1 << 25) // (kv * dim * groups * seqs))))
    return dict(op=op, groups=groups, seqs=seqs, prefix=prefix, longest=longest, q_heads=heads, kv_heads=kv,
                head_dim=dim, page=page, dtype=rng.choice(["bf16", "bf16", "bf16", "int8", "f32"]))


def _lengths(case):
    """Slots of each sequence, past the prefix where there is one; a rule of
    the case alone. A batch of 8 or more sequences has an empty one."""
    n, longest = case.get("groups", 1) * case["seqs"], case["longest"]
    lens = [longest] + [1 + int((longest - 1) * ((0.618034 * i) % 1.0)) for i in range(1, n)]
    return [0 if n >= 8 and i == n // 2 else v for i, v in enumerate(lens)]


def _slot_bytes(case):
    """Of one slot's key and value of one head, a scale beside each in 8 bits."""
    d = case["head_dim"]
    return 2 * {"f32": 4 * d, "bf16": 2 * d, "int8": d + 4}[case.get("dtype", "int8")]


def work(case):
    if case["op"] in ("logprobs", "logprobs_grad"):
        t, v = case["rows"], case["vocab"]
        if case["op"] == "logprobs":
            return dict(bytes=4 * t * v + 4 * t * (5 + 2 * case["top"]), flops=5 * t * v)
        return dict(bytes=8 * t * v + 4 * t * (6 if case["entropy"] else 4), flops=(8 if case["entropy"] else 4) * t * v)
    lens, kv, d, slot = _lengths(case), case["kv_heads"], case["head_dim"], _slot_bytes(case)
    if case["op"] == "write_read":
        total, fresh = sum(lens), sum(min(n, case["fresh"]) for n in lens)
        return dict(bytes=kv * (fresh + total) * (slot + 8 * d), flops=kv * d * (6 * fresh + 2 * total))
    heads, n, slots = case["q_heads"], len(lens), sum(lens)
    if case["op"] == "shared":
        shared = case["prefix"]
        return dict(bytes=kv * slot * (slots + case["groups"] * shared) + 8 * n * heads * d,
                    flops=4 * heads * d * (slots + n * shared))
    return dict(bytes=kv * slot * slots + 8 * n * heads * d, flops=4 * heads * d * slots)


# ------------------------------------------------------------------ inputs --
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)


def _quantised(x):
    """(codes, scale) of rows of float32, the codes by real arithmetic."""
    top = x.abs().amax(-1, keepdim=True)
    exactly = 127.0 * x.double() / top.double().clamp_min(1e-300)
    return torch.round(exactly).clamp(-127, 127).to(torch.int8), (top.double() / 127).float()


def _logits(case, seed):
    """Rows from nearly flat to sharply peaked; the last 1/64 of the vocabulary
    is padding and masked, and one row in 16 is a padded one."""
    g = _generator(seed)
    t, v = case["rows"], case["vocab"]
    x = torch.randn(t, v, generator=g, device="cuda")
    x *= 0.5 + 4 * torch.rand(t, 1, generator=g, device="cuda")
    live = v - v // 64
    x[:, live:] = float("-inf")
    tokens = torch.randint(0, live, (t,), generator=g, device="cuda")
    # Half of the rows ask for a likely token, as a sampler or a trained model does.
    likely = torch.arange(t, device="cuda") % 2 == 0
    tokens = torch.where(likely, x[:, :max(1, live // 50)].argmax(-1), tokens)
    padded = torch.arange(t, device="cuda") % 16 == 15
    s = dict(case=case, logits=x, tokens=torch.where(padded, -1, tokens).float())
    if case["op"] == "logprobs_grad":
        s["d_logprobs"] = torch.randn(t, generator=g, device="cuda")
        s["d_entropy"] = 0.1 * torch.randn(t, generator=g, device="cuda")
    return s


def _cache_inputs(case, seed):
    """Pools, page tables in random order and lengths. Where sequences share a
    prefix, its pages come first in each of their tables."""
    g = _generator(seed)
    lens, page, kv, d = _lengths(case), case["page"], case["kv_heads"], case["head_dim"]
    groups, dtype = case.get("groups", 1), case.get("dtype", "int8")
    before = case.get("prefix", 0) // page
    counts = [-(-n // page) for n in lens]
    pages = groups * before + sum(counts) + 3
    order = torch.randperm(pages, generator=g, device="cuda").cpu().numpy()
    table = np.zeros((len(lens), max(1, before + max(counts))), dtype=np.int32)
    at = groups * before
    for i, c in enumerate(counts):
        first = i // case["seqs"] * before
        table[i, :before] = order[first:first + before]
        table[i, before:before + c] = order[at:at + c]
        at += c
    s = dict(case=case, lens=[n + case.get("prefix", 0) for n in lens], table=table, pages=pages)
    for name in ("k", "v"):
        x = torch.randn(pages, kv, page, d, generator=g, device="cuda")
        # Channels of a key differ in size; a value's rows do.
        x *= torch.rand((kv, 1, d) if name == "k" else (pages, kv, page, 1), generator=g, device="cuda") + 0.5
        if dtype == "int8":
            s[name], s[name + "_scale"] = _quantised(x)
        else:
            s[name] = x.to(torch.bfloat16) if dtype == "bf16" else x
    if case["op"] == "write_read":
        fresh = sum(min(n, case["fresh"]) for n in lens)
        # Keys and values side by side, as a fused projection leaves them.
        s["heads"] = torch.randn(fresh, 2 * kv, d, generator=g, device="cuda")
        s["heads"] *= torch.rand(fresh, 2 * kv, 1, generator=g, device="cuda") + 0.1
    else:
        s["q"] = 1.5 * torch.randn(len(lens), case["q_heads"], d, generator=g, device="cuda")
    return s


def prepare(case, seed):
    """What a program holds before the call. Of the framework (`own`) that is
    its tensors, its cache and the batch's page tables; the same values."""
    if case["op"] in ("logprobs", "logprobs_grad"):
        s = _logits(case, seed)
        if case["op"] == "logprobs_grad":  # the forward pass came before
            _, s["entropy"], s["norm"] = _logprobs(s["logits"], s["tokens"])
        if own:
            from porch_b200 import api

            s = dict(case=case, **{k: api.tensor_from_device(v) for k, v in s.items() if k != "case"})
        return s
    s = _cache_inputs(case, seed)
    fresh = [min(n, case["fresh"]) for n in s["lens"]] if case["op"] == "write_read" else None
    if own:
        from porch_b200 import api

        cache = api.KVCache(s["pages"], case["page"], case["kv_heads"], case["head_dim"],
                            dtype=case.get("dtype", "int8"))
        for pool, name in zip(cache.pools(), ("k", "v")):
            pool = torch.as_tensor(pool, device="cuda")
            (pool.view(torch.bfloat16) if s[name].dtype == torch.bfloat16 else pool).copy_(s[name])
        if "k_scale" in s:
            for pool, name in zip(cache.scales(), ("k_scale", "v_scale")):
                torch.as_tensor(pool, device="cuda").copy_(s[name][..., 0])
        torch.cuda.synchronize()
        prefix = [case["prefix"]] * len(s["lens"]) if case["op"] == "shared" else None
        mine = dict(case=case, cache=cache, batch=cache.batch(s["table"], s["lens"], appended=fresh, prefix=prefix))
        if case["op"] == "write_read":
            heads, kv = api.tensor_from_device(s["heads"]), case["kv_heads"]
            mine["new"] = [api.materialize(heads[api.all, i * kv:(i + 1) * kv, api.all]) for i in (0, 1)]
        else:
            mine["q"] = api.tensor_from_device(s["q"])
        return mine
    # The rows of the pools that the sequences' slots are, in their order.
    at = [(np.repeat(row[:-(-n // case["page"])].astype(np.int64), case["page"])[:n], np.arange(n) % case["page"])
          for row, n in zip(s["table"], s["lens"])]
    if fresh is not None:
        s["slots"] = tuple(torch.from_numpy(np.concatenate(x)).cuda() for x in zip(*at))
        s["new_slots"] = tuple(torch.from_numpy(np.concatenate([y[len(y) - f:] for y, f in zip(x, fresh)])).cuda()
                               for x in zip(*at))
    s["length"] = torch.tensor(s["lens"], device="cuda") - case.get("prefix", 0)
    s["table"] = torch.from_numpy(s["table"]).cuda().long()
    return s


# --------------------------------------------------------------- plain form --
def _logprobs(x, tokens):
    top = x.amax(-1, keepdim=True)
    rel = x - top
    e = torch.exp(rel)
    total = e.sum(-1, dtype=torch.float64)
    weighted = (e * torch.where(e > 0, rel, 0.0)).sum(-1, dtype=torch.float64)
    entropy = (total.log() - weighted / total).float()
    at = tokens.long()
    said = (rel.gather(-1, at.clamp_min(0)[:, None])[:, 0].double() - total.log()).float()
    return torch.where(at >= 0, said, 0.0), entropy, torch.stack((top[:, 0], total.float()), -1)


def _grad(s):
    x, at, entropy = s["logits"], s["tokens"].long(), s["case"]["entropy"]
    rel = x - s["norm"][:, :1]
    p = torch.exp(rel) / s["norm"][:, 1:]
    g = torch.where(at >= 0, s["d_logprobs"], 0.0)[:, None]
    d = -g * p
    d.scatter_add_(-1, at.clamp_min(0)[:, None], g)
    if entropy:
        logp = torch.where(p > 0, rel - s["norm"][:, 1:].log(), 0.0)
        d -= s["d_entropy"][:, None] * p * (logp + s["entropy"][:, None])
    return d


def _values(s, name, pages):
    """The values of these pages' slots in 32 bits, [..., heads, slots, head_dim]."""
    x = s[name][pages].float()
    if name + "_scale" in s:
        x = x * s[name + "_scale"][pages]
    return x.transpose(-4, -3).flatten(-3, -2)


def _attend(s):
    case = s["case"]
    groups, kv, d = case.get("groups", 1), case["kv_heads"], case["head_dim"]
    n, before = len(s["lens"]), case.get("prefix", 0) // case["page"]
    own_pages = s["table"][:, before:] if s["table"].shape[1] > before else s["table"][:, :1]
    k, v = _values(s, "k", own_pages), _values(s, "v", own_pages)  # [sequences, heads, slots, D]
    q = s["q"].view(n, kv, -1, d) * d ** -0.5
    seen = torch.arange(k.shape[2], device="cuda") < s["length"][:, None]
    logits = (q @ k.transpose(-1, -2)).masked_fill(~seen[:, None, None], float("-inf"))
    v = v.masked_fill(~seen[:, None, :, None], 0.0)
    if before:
        shared = s["table"][::case["seqs"], :before]  # of each group
        kp, vp = _values(s, "k", shared), _values(s, "v", shared)  # [groups, heads, slots, D]
        per = q.shape[2]
        qg = q.view(groups, -1, kv, per, d).transpose(1, 2).flatten(2, 3)  # [groups, heads, sequences x per, D]
        first = (qg @ kp.transpose(-1, -2)).unflatten(2, (-1, per)).transpose(1, 2).flatten(0, 1)
        logits = torch.cat((first, logits), -1)
    top = logits.amax(-1, keepdim=True).clamp_min(-3.0e38)
    p = torch.exp(logits - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    if not before:
        return (p @ v).reshape(n, -1, d)
    slots = case["prefix"]
    pg = p[..., :slots].view(groups, -1, kv, per, slots).transpose(1, 2).flatten(2, 3)
    first = (pg @ vp).unflatten(2, (-1, per)).transpose(1, 2).flatten(0, 1)
    return (first + p[..., slots:] @ v).reshape(n, -1, d)


def _write_read(s):
    kv = s["case"]["kv_heads"]
    page, place = s["new_slots"]
    s["k"][page, :, place], s["k_scale"][page, :, place] = _quantised(s["heads"][:, :kv])
    s["v"][page, :, place], s["v_scale"][page, :, place] = _quantised(s["heads"][:, kv:])
    page, place = s["slots"]
    return (s["k"][page, :, place].float() * s["k_scale"][page, :, place],
            s["v"][page, :, place].float() * s["v_scale"][page, :, place])


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        return _run_own(s, case, op)
    if op == "logprobs_grad":
        return _grad(s)
    if op == "write_read":
        return _write_read(s)
    if op != "logprobs":
        return _attend(s)
    said, entropy, norm = _logprobs(s["logits"], s["tokens"])
    if not case["top"]:
        return said, entropy, norm
    value, token = torch.sort(s["logits"], dim=-1, descending=True, stable=True)
    value, token = value[:, :case["top"]], token[:, :case["top"]]
    return said, entropy, norm, (value - norm[:, :1]) - norm[:, 1:].log(), token.float()


def _run_own(s, case, op):
    from porch_b200 import api

    if op == "logprobs":
        out = api.token_logprobs(s["logits"], s["tokens"], top=case["top"])
    elif op == "logprobs_grad":
        more = dict(d_entropy=s["d_entropy"], entropy=s["entropy"]) if case["entropy"] else {}
        out = (api.token_logprobs_backward(s["d_logprobs"], s["logits"], s["tokens"], s["norm"], **more),)
    elif op == "write_read":
        s["batch"].append(*s["new"])
        out = s["batch"].read()
    else:
        out = (api.paged_attention(s["q"], s["batch"]),)
    seen = tuple(torch.as_tensor(t, device="cuda") for t in out)
    return seen if len(seen) > 1 else seen[0]


# ------------------------------------------------------------------ 64 bits --
def exact(case, seed):
    if case["op"] in ("logprobs", "logprobs_grad"):
        return _exact_logprobs(case, seed)
    if case["op"] == "write_read":
        return _exact_write_read(case, seed)
    return _exact_attend(case, seed)


def _exact_logprobs(case, seed):
    s = _logits(case, seed)
    parts = [[] for _ in range(5)]
    for i in range(0, case["rows"], 256):  # a few rows at a time: 64 bits take room
        x, at = s["logits"][i:i + 256].double(), s["tokens"][i:i + 256].long()
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
        if case["op"] == "logprobs_grad":
            hot = torch.nn.functional.one_hot(at.clamp_min(0), x.shape[1]) * (at >= 0)[:, None]
            d = s["d_logprobs"][i:i + 256].double()[:, None] * (hot - p * (at >= 0)[:, None])
            if case["entropy"]:
                bonus = torch.where(p > 0, p * (logp + entropy[:, None]), 0.0)
                d = d - s["d_entropy"][i:i + 256].double()[:, None] * bonus
            parts[0].append(d)
            continue
        parts[0].append(torch.where(at >= 0, logp.gather(-1, at.clamp_min(0)[:, None])[:, 0], 0.0))
        parts[1].append(entropy)
        top = x.max(-1).values
        parts[2].append(torch.stack((top, (torch.logsumexp(x, -1) - top).exp()), -1))
        if case["top"]:
            order = torch.argsort(-s["logits"][i:i + 256], dim=-1, stable=True)[:, :case["top"]]
            parts[3].append(logp.gather(-1, order))
            parts[4].append(order.double())
    out = tuple(torch.cat(x) for x in parts if x)
    return out if len(out) > 1 else out[0]


def _exact_write_read(case, seed):
    s = _cache_inputs(case, seed)
    kv, page = case["kv_heads"], case["page"]
    out, at = ([], []), 0
    for i, n in enumerate(s["lens"]):
        fresh = min(n, case["fresh"])
        slot = torch.arange(n, device="cuda")
        pages = torch.from_numpy(s["table"][i]).cuda().long()[slot // page]
        new = s["heads"][at:at + fresh].double()
        at += fresh
        for j, name in enumerate(("k", "v")):
            x = s[name][pages, :, slot % page].double() * s[name + "_scale"][pages, :, slot % page].double()
            y = new[:, j * kv:(j + 1) * kv]
            unit = y.abs().max(-1, keepdim=True).values
            # Integers divide without a remainder where a value lies on a border.
            x[n - fresh:] = torch.round(y * 127 / unit) * (unit / 127)
            out[j].append(x)
    return tuple(torch.cat(x) for x in out)


def _exact_attend(case, seed):
    s = _cache_inputs(case, seed)
    kv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(len(s["lens"]), case["q_heads"], d, dtype=torch.float64, device="cuda")
    if len(s["lens"]) * sum(s["lens"]) * kv > 1 << 33:
        return None
    for i, n in enumerate(s["lens"]):
        if n == 0:
            continue
        at = torch.from_numpy(s["table"][i, :-(-n // page)]).cuda().long()
        k, v = (s[name][at].double() * (s[name + "_scale"][at].double() if name + "_scale" in s else 1)
                for name in ("k", "v"))
        k, v = (x.transpose(0, 1).reshape(kv, -1, d)[:, :n] for x in (k, v))
        q = s["q"][i].unflatten(0, (kv, -1)).double()
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(d), -1)
        out[i] = torch.einsum("hgn,hnd->hgd", p, v).flatten(0, 1)
    return out
