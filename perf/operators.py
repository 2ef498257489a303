"""A serving step's operators around a shared prompt and drafted tokens, as
cases that can be timed, in plain torch and through the framework's calls.

The kinds of case ("call"):
  norm    qk_norm_rope_store_kv: per-head RMSNorm of q and k, RoPE and the
          paged K/V store from the stacked projection rows
  prefix  shared_prefix_attention: attention of sequences whose block tables
          begin with the same blocks (one or several groups of them)
  verify  verify_drafts: drafted tokens accepted or resampled against the
          target's logits

A case is a dict of plain values; prepare(case, seed) makes on the GPU what a
serving program has in hand before the call, run(state) makes one pass and
returns every output, and exact(case, seed) is the same function in 64 bits.
Where `own` is false, run computes the operator from elementary torch
operations instead of the framework's kernels. Sequence lengths are part of a
case (drawn from its "lengths" number), values come from the seed.
"""
from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parent.parent
own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "none": 0}
MAX_POS = 20480
EPS = 1e-6


@functools.lru_cache(maxsize=1)
def _kernels():
    if str(ROOT / "llm-engine_amd") not in sys.path:
        sys.path.insert(0, str(ROOT / "llm-engine_amd"))
    from llm_engine_amd import kernels
    return kernels


# ---- the cases ----
def _norm(name, heads, rows, act="bf16", kv="bf16", bias=False):
    c = dict(call="norm", q_heads=heads[0], kv_heads=heads[1], head_dim=heads[2], rows=rows, act=act, kv=kv, bias=bias)
    return dict(c, name=name) if name else c


def _prefix(name, heads, groups, seqs, prefix, suffix, rows=1, act="bf16", kv="bf16", block=16, lengths=1):
    """groups x seqs sequences; a group's tables begin with the same prefix // block blocks. suffix: a sequence's own
    keys beyond them, the step's 1 to `rows` rows (the sampled token and its drafts) among them."""
    c = dict(call="prefix", q_heads=heads[0], kv_heads=heads[1], head_dim=heads[2], groups=groups, seqs=seqs,
             prefix=prefix // block * block, suffix_lo=suffix[0], suffix_hi=suffix[1], rows=rows, act=act, kv=kv,
             block=block, lengths=lengths)
    return dict(c, name=name) if name else c


def _verify(name, seqs, drafts, vocab, logits="f32", probs="f32", greedy=0.0, lengths=1):
    """seqs sequences of 1 to `drafts` drafted tokens (0: none); `greedy` of them at temperature 0. probs "none": the
    drafts come from a lookup, without probabilities."""
    c = dict(call="verify", seqs=seqs, drafts=drafts, vocab=vocab, logits=logits, probs=probs, greedy=greedy,
             lengths=lengths)
    return dict(c, name=name) if name else c


def listed():
    qwen, llama, wide = (14, 2, 64), (32, 4, 64), (32, 8, 128)  # Qwen2.5-0.5B, TinyLlama-1.1B, a head_dim-128 GQA-4 shape
    return [
        # One user's decode step: one row, where only latency counts.
        _norm("norm_one", qwen, 1),
        # A full batch with four drafts each: 64 sequences x 5 rows.
        _norm("norm_decode", wide, 320),
        # The fp32 engine's odd-sized step, with the projection's bias.
        _norm("norm_f32", qwen, 777, act="f32", kv="f32", bias=True),
        # The scheduler's default budget of prefill tokens in one step.
        _norm("norm_prefill", wide, 4096),
        # A few users behind one short system prompt.
        _prefix("prefix_small", qwen, 1, 4, 512, (8, 100), lengths=2),
        # A running batch behind one long prompt, one row each.
        _prefix("prefix_decode", qwen, 1, 64, 4096, (16, 512), lengths=3),
        # Three agents' prompts, 16 sequences each, up to four drafts beside the sampled token, fp16.
        _prefix("prefix_drafts", wide, 3, 16, 2000, (5, 700), rows=5, act="f16", kv="f16", lengths=4),
        # The fp32 engine's batch.
        _prefix("prefix_f32", qwen, 1, 24, 1500, (1, 300), act="f32", kv="f32", lengths=5),
        # One document read by 256 samples: the compute-bound end.
        _prefix("prefix_long", wide, 1, 256, 16384, (64, 1024), lengths=6),
        # One user's four drafts over the smaller vocabulary.
        _verify("verify_one", 1, 4, 32000, lengths=7),
        # A full batch over the largest vocabulary of the configurations, a quarter of it greedy.
        _verify("verify_batch", 64, 5, 151936, greedy=0.25, lengths=8),
        # Lookup drafts without probabilities, 16-bit logits.
        _verify("verify_lookup", 32, 8, 151936, logits="bf16", probs="none", lengths=9),
    ]


HEADS = [(14, 2, 64), (32, 4, 64), (32, 8, 128), (12, 12, 64), (28, 4, 128), (10, 10, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: 1 to 4096 rows through the norms; 1 to 4 groups of 1 to 256 sequences behind 8
    to 16384 shared keys with 1 to 1024 of their own and 1 to 8 rows; 1 to 64 sequences of 0 to 8 drafts over 1000 to
    151936 tokens; every type, block sizes 8 to 64."""
    call = rng.choice(["norm", "prefix", "prefix", "verify"])
    if call == "norm":
        heads, kv = rng.choice(HEADS), rng.choice(["bf16", "bf16", "f16", "f32"])
        return _norm(None, heads, _log(rng, 1, 4096), act=rng.choice([kv, kv, "f32"]), kv=kv, bias=rng.random() < 0.3)
    if call == "verify":
        return _verify(None, _log(rng, 1, 64), rng.choice([0, 1, 2, 3, 4, 5, 6, 7, 8]), _log(rng, 1000, 151936),
                       logits=rng.choice(["f32", "f32", "bf16", "f16"]), probs=rng.choice(["f32", "f32", "bf16", "none"]),
                       greedy=rng.choice([0.0, 0.0, 0.3, 1.0]), lengths=rng.randrange(1 << 20))
    limit = max(_cost(c) for c in listed() if c["call"] == "prefix")
    for _ in range(64):
        kv = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
        block = rng.choice([16, 16, 16, 8, 32, 64])
        hi = _log(rng, 1, 1024)
        rows = rng.choice([1, 1, 2, 4, 5, 8])
        c = _prefix(None, rng.choice(HEADS), rng.choice([1, 1, 1, 2, 3, 4]), _log(rng, 1, 256),
                    max(block, _log(rng, 16, 16384)), (rng.choice([1, max(1, hi // 8), hi]), hi), rows=rows,
                    act=rng.choice([kv, kv, kv, "f32"]), kv=kv, block=block, lengths=rng.randrange(1 << 20))
        if c["groups"] * c["seqs"] <= 256 and _cost(c) <= limit:
            return c
    return _prefix(None, (14, 2, 64), 1, 7, 333, (1, 77), lengths=rng.randrange(1 << 20))


def _cost(c):
    w = work(c)
    return w["bytes"] / 2e12 + w["flops"] / (0.2e15 if c["kv"] != "f32" and c["act"] == c["kv"] else 0.03e15)


# ---- lengths: part of the case ----
def _spans(c):
    """Own keys and rows of every sequence of a prefix case; a sequence's rows are its last keys."""
    rng = np.random.default_rng(c["lengths"])
    n = c["groups"] * c["seqs"]
    own_keys = rng.integers(c["suffix_lo"], c["suffix_hi"] + 1, n)
    return own_keys, np.minimum(rng.integers(1, c["rows"] + 1, n), own_keys)


def _drafts(c):
    rng = np.random.default_rng(c["lengths"])
    n = np.zeros(c["seqs"], dtype=np.int64) if c["drafts"] == 0 else rng.integers(1, c["drafts"] + 1, c["seqs"])
    return n, rng.random(c["seqs"]) < c["greedy"]


def work(case):
    c = case
    if c["call"] == "verify":
        n, _ = _drafts(c)
        rows = int(n.sum()) + c["seqs"]
        # every target row once, and one row of draft probabilities a sequence
        return {"bytes": c["vocab"] * (rows * SIZE[c["logits"]] + c["seqs"] * SIZE[c["probs"]]) + 16 * rows,
                "flops": 4 * rows * c["vocab"]}
    H, KH, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    if c["call"] == "norm":
        n = c["rows"]
        return {"bytes": n * ((2 * H + 2 * KH) * d * SIZE[c["act"]] + 2 * KH * d * SIZE[c["kv"]] + 4 * d + 8),
                "flops": 9 * n * (H + KH) * d}
    keys, rows = _spans(c)
    n = int(rows.sum())
    pairs = int((rows * (c["prefix"] + keys - rows) + rows * (rows + 1) // 2).sum())
    kv_rows = c["groups"] * c["prefix"] + int(keys.sum())  # the shared ones once a group
    return {"bytes": kv_rows * KH * d * 2 * SIZE[c["kv"]] + 2 * n * H * d * SIZE[c["act"]], "flops": 4 * H * d * pairs}


def _rand(seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return dev, g


# ---- per-head norms, rotation and the K/V store ----
def _prepare_norm(c, seed):
    dev, g = _rand(seed)
    n, H, KH, d = c["rows"], c["q_heads"], c["kv_heads"], c["head_dim"]
    act, kv = DTYPES[c["act"]], DTYPES[c["kv"]]
    pool = (n + 15) // 16 * 16 + 64

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    inv = 1e6 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
    ang = torch.arange(MAX_POS, device=dev, dtype=torch.float64)[:, None] * inv
    return dict(case=c, qkv=(1.5 * normal(n, (H + 2 * KH) * d)).to(act),
                bias=0.5 * normal((H + 2 * KH) * d) if c["bias"] else None,
                q_norm=1 + 0.2 * normal(d), k_norm=1 + 0.2 * normal(d), cos=ang.cos().float(), sin=ang.sin().float(),
                positions=torch.randint(0, MAX_POS, (n,), device=dev, generator=g, dtype=torch.int32),
                slots=torch.randperm(pool, device=dev, generator=g)[:n].to(torch.int32),
                k=normal(pool, KH * d).to(kv), v=normal(pool, KH * d).to(kv),
                q=torch.empty(n, H * d, device=dev, dtype=act))


def _run_norm(s):
    c = s["case"]
    H, KH, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    if own:
        _kernels().qk_norm_rope_store_kv(s["qkv"], s["positions"], s["slots"], s["cos"], s["sin"], s["q_norm"],
                                         s["k_norm"], EPS, H, KH, d, s["k"], s["v"], bias=s["bias"], q_out=s["q"])
        return [s["q"], s["k"], s["v"]]
    x = s["qkv"].float()
    if s["bias"] is not None:
        x = x + s["bias"]
    x = x.reshape(-1, H + 2 * KH, d)
    w = torch.cat([s["q_norm"].expand(H, d), s["k_norm"].expand(KH, d)])
    y = x[:, :H + KH]
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    a, b = y[..., :d // 2], y[..., d // 2:]
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    slots = s["slots"].long()
    s["q"].copy_(y[:, :H].reshape(-1, H * d))
    s["k"][slots] = y[:, H:].reshape(-1, KH * d).to(s["k"].dtype)
    s["v"][slots] = x[:, H + KH:].reshape(-1, KH * d).to(s["v"].dtype)
    return [s["q"], s["k"], s["v"]]


def _exact_norm(c, seed):
    s = _prepare_norm(c, seed)
    H, KH, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"].double() + (0 if s["bias"] is None else s["bias"].double())
    q, k, v = x.split([H * d, KH * d, KH * d], dim=-1)
    cos, sin = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]

    def head(x, w):
        n = w.double() * x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt()
        lo, hi = n.chunk(2, dim=-1)
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], dim=-1)

    kc, vc, at = s["k"].double(), s["v"].double(), s["slots"].long()
    kc[at] = torch.cat([head(k[:, i * d:(i + 1) * d], s["k_norm"]) for i in range(KH)], dim=-1)
    vc[at] = v
    return [torch.cat([head(q[:, i * d:(i + 1) * d], s["q_norm"]) for i in range(H)], dim=-1), kc, vc]


# ---- attention behind shared prefixes ----
def _tables(c, seed):
    """Block tables [sequences, blocks] (padded with 0) from a permuted pool, a group's prefix blocks alike; the
    sequences' key counts and rows; the pool's size."""
    keys, rows = _spans(c)
    n, pb = len(keys), c["prefix"] // c["block"]
    sb = -(-keys // c["block"])
    used = c["groups"] * pb + int(sb.sum())
    ids = np.random.default_rng(seed).permutation(used + 16)[:used].astype(np.int32)
    tables = np.zeros((n, pb + int(sb.max())), dtype=np.int32)
    tables[:, :pb] = np.repeat(ids[:c["groups"] * pb].reshape(c["groups"], pb), c["seqs"], axis=0)
    valid = np.arange(int(sb.max()))[None] < sb[:, None]
    tables[:, pb:][valid] = ids[c["groups"] * pb:]
    return tables, pb + sb, keys + c["prefix"], rows, used + 16


def _prepare_prefix(c, seed):
    dev, g = _rand(seed)
    H, KH, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    tables, blocks, keys, rows, pool = _tables(c, seed)
    n = int(rows.sum())
    act, kv = DTYPES[c["act"]], DTYPES[c["kv"]]

    def normal(*shape, dtype):
        return torch.randn(*shape, device=dev, generator=g).to(dtype)

    seq = np.repeat(np.arange(len(rows)), rows)
    first = np.cumsum(rows) - rows
    pos = np.arange(n) - first[seq] + (keys - rows)[seq]
    # a group's rows, padded to the widest group, and where each row stands among them
    per = rows.reshape(c["groups"], c["seqs"]).sum(1)
    start, most = np.cumsum(per) - per, int(per.max())
    grid = np.minimum(start[:, None] + np.arange(most), n - 1)
    place = (seq // c["seqs"]) * most + np.arange(n) - start[seq // c["seqs"]]
    s = dict(case=c, q=normal(n, H * d, dtype=act), k=normal(pool * c["block"], KH * d, dtype=kv),
             v=normal(pool * c["block"], KH * d, dtype=kv), out=torch.empty(n, H * d, device=dev, dtype=act),
             scale=1.0 / math.sqrt(d), tables=torch.from_numpy(tables).to(dev).long(),
             seq=torch.from_numpy(seq).to(dev), pos=torch.from_numpy(pos).to(dev),
             grid=torch.from_numpy(grid).to(dev), place=torch.from_numpy(place).to(dev))
    if own:  # the packed step, as a program keeps it for all of its layers
        kernels = _kernels()
        none = np.zeros(int(keys.max()), dtype=np.int32)
        slices = [kernels.Slice(i, int(keys[i] - rows[i]), int(rows[i]), True, tables[i, :blocks[i]], none[:keys[i]])
                  for i in range(len(rows))]
        s["plan"] = kernels.PrefixPlan(slices, H, KH, d, c["block"], kv).upload()
        s["ws"] = kernels.new_workspace(s["plan"].workspace_size(), dev)
    return s


def _run_prefix(s):
    c = s["case"]
    if own:
        return _kernels().shared_prefix_attention(s["q"], s["k"], s["v"], s["plan"], s["scale"], out=s["out"],
                                                  workspace=s["ws"])
    H, KH, d, P, bs = c["q_heads"], c["kv_heads"], c["head_dim"], c["prefix"], c["block"]
    G, n, pb = H // KH, s["q"].shape[0], P // bs
    k, v = s["k"].reshape(-1, bs, KH, d), s["v"].reshape(-1, bs, KH, d)
    # scores against the shared keys, a group's rows together: [groups, KH, rows x G, P]
    shared = s["tables"][::c["seqs"], :pb]
    kp, vp = (t[shared].float().reshape(c["groups"], P, KH, d).permute(0, 2, 1, 3).contiguous() for t in (k, v))
    q = s["q"].float().reshape(n, KH, G, d)
    most = s["grid"].shape[1]
    qg = q[s["grid"]].permute(0, 2, 1, 3, 4).reshape(c["groups"], KH, most * G, d)
    sp = torch.matmul(qg, kp.transpose(2, 3).contiguous()) * s["scale"]
    # against each row's own keys: [rows, KH, G, S]
    mine = s["tables"][:, pb:][s["seq"]]
    S = mine.shape[1] * bs
    ks, vs = (t[mine].float().reshape(n, S, KH, d).permute(0, 2, 1, 3).contiguous() for t in (k, v))
    ss = torch.matmul(q, ks.transpose(2, 3).contiguous()) * s["scale"]
    hidden = P + torch.arange(S, device=ss.device)[None] > s["pos"][:, None]
    ss = ss.masked_fill(hidden[:, None, None], -math.inf)
    vs = vs.masked_fill(hidden[:, None, :, None], 0.0)

    def rows(x):  # from the groups' layout to a row's: [rows, KH, G, last]
        x = x.reshape(c["groups"], KH, most, G, -1).permute(0, 2, 1, 3, 4).reshape(c["groups"] * most, KH, G, -1)
        return x[s["place"]]

    mp = sp.amax(-1, keepdim=True)
    sp = torch.exp(sp - mp)
    ms = ss.amax(-1, keepdim=True)
    ss = torch.exp(ss - ms)
    lp, op, mp = rows(sp.sum(-1, keepdim=True)), rows(torch.matmul(sp, vp)), rows(mp)
    ls, os_ = ss.sum(-1, keepdim=True), torch.matmul(ss, vs)
    m = torch.maximum(mp, ms)
    a, b = torch.exp(mp - m), torch.exp(ms - m)
    s["out"].copy_(((op * a + os_ * b) / (lp * a + ls * b)).reshape(n, H * d))
    return s["out"]


def _exact_prefix(c, seed):
    if work(c)["flops"] > 2e11:
        return None
    s = _prepare_prefix(c, seed)
    tables, _, keys, rows, _ = _tables(c, seed)
    H, KH, d, bs = c["q_heads"], c["kv_heads"], c["head_dim"], c["block"]
    out, r = torch.empty(len(s["seq"]), H, d, device=s["q"].device, dtype=torch.float64), 0
    for t, m, w in zip(s["tables"], keys.tolist(), rows.tolist()):
        at = (t[:, None] * bs + torch.arange(bs, device=t.device)).reshape(-1)[:m]
        q = s["q"][r:r + w].double().reshape(w, H, d)
        late = torch.arange(m, device=t.device)[None] > torch.arange(m - w, m, device=t.device)[:, None]
        for j in range(KH):
            kk, vv = (x[at, j * d:(j + 1) * d].double() for x in (s["k"], s["v"]))
            for h in range(j * (H // KH), (j + 1) * (H // KH)):
                p = torch.softmax(((q[:, h] @ kk.T.contiguous()) * s["scale"]).masked_fill(late, -math.inf), dim=-1)
                out[r:r + w, h] = p @ vv
        r += w
    return out.reshape(len(s["seq"]), H * d)


# ---- verification of drafted tokens ----
def _prepare_verify(c, seed):
    dev, g = _rand(seed)
    n, greedy = _drafts(c)
    cu = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    N, V, S = int(n.sum()), c["vocab"], c["seqs"]

    def uniform(k):
        return torch.rand(k, device=dev, generator=g)

    seq = torch.from_numpy(np.repeat(np.arange(S), n)).to(dev)
    temperature = (0.5 + uniform(S)) * torch.from_numpy(~greedy).to(dev)
    logits = (4 * torch.randn(N + S, V, device=dev, generator=g)).to(DTYPES[c["logits"]])
    # the draft model: near the target, a temperature of its own, its tokens sampled from what it says
    near = logits[torch.arange(N, device=dev) + seq].float() + torch.randn(N, V, device=dev, generator=g)
    q = torch.softmax(near / torch.where(temperature > 0, temperature, 0.25)[seq][:, None], dim=-1)
    tokens = (torch.log(q) - torch.log(-torch.log(torch.rand(N, V, device=dev, generator=g).clamp(1e-12, 1 - 1e-7))))
    tokens = tokens.argmax(-1).to(torch.int32) if N else torch.zeros(0, device=dev, dtype=torch.int32)
    s = dict(case=c, logits=logits, cu=torch.from_numpy(cu).to(dev), tokens=tokens,
             probs=None if c["probs"] == "none" else q.to(DTYPES[c["probs"]]), temperature=temperature,
             accept_u=uniform(N), sample_u=uniform(S))
    if own:
        kernels = _kernels()
        s["out"] = torch.empty(S, c["drafts"] + 1, device=dev, dtype=torch.int32)
        s["accepted"] = torch.empty(S, device=dev, dtype=torch.int32)
        s["ws"] = kernels.new_workspace(kernels.verify_drafts_workspace_size(S, N, V), dev)
    return s


def _run_verify(s):
    c = s["case"]
    if own:
        return _kernels().verify_drafts(s["logits"], s["cu"], s["tokens"], s["accept_u"], s["sample_u"], c["drafts"],
                                        draft_probs=s["probs"], temperature=s["temperature"], out=s["out"],
                                        n_accepted=s["accepted"], workspace=s["ws"])
    S, D, V, dev = c["seqs"], c["drafts"], c["vocab"], s["logits"].device
    cu, N = s["cu"].long(), s["tokens"].numel()
    row = torch.arange(N + S, device=dev)
    # a target row's sequence: rows cu[s] + s to cu[s + 1] + s
    seq = torch.searchsorted(cu[1:] + torch.arange(S, device=dev), row)
    x, t = s["logits"].double(), s["temperature"].double()[seq][:, None]
    top = x.amax(-1, keepdim=True)
    ids = torch.arange(V, device=dev)
    best = torch.where(x == top, ids, V).amin(-1, keepdim=True)
    w = torch.where(t > 0, torch.exp((x - top) / torch.where(t > 0, t, 1.0)), (ids == best).double())
    p = w / w.sum(-1, keepdim=True)
    # accepted drafts: the leading ones with u q(x) < p(x)
    at, place = cu[:-1, None] + torch.arange(D, device=dev), torch.arange(D, device=dev)
    there = at < cu[1:, None]
    at = torch.where(there, at, 0)
    pad = torch.full((S, 1), -1, device=dev, dtype=torch.int32)
    if N:
        draft = s["tokens"].long()
        i = torch.arange(N, device=dev)
        q_at = 1.0 if s["probs"] is None else s["probs"][i, draft].double()
        good = s["accept_u"].double() * q_at < p[i + torch.searchsorted(cu[1:], i, right=True), draft]
        n_acc = (good[at] & there).long().cumprod(-1).sum(-1)
    else:
        n_acc = torch.zeros(S, device=dev, dtype=torch.int64)
    # the next token: from max(p - q, 0) of the rejected row, or from p after the last draft
    last = cu[:-1] + n_acc
    base = p[last + torch.arange(S, device=dev)]
    left = base
    if N:
        rejected = (last < cu[1:])[:, None]
        at_last = torch.where(last < cu[1:], last, 0)
        q = torch.zeros_like(base) if s["probs"] is None else s["probs"][at_last].double()
        if s["probs"] is None:
            q = (ids == draft[at_last][:, None]).double()
        left = torch.where(rejected, (base - q).clamp(min=0), base)
        left = torch.where((left.sum(-1, keepdim=True) > 0) & (s["temperature"] > 0)[:, None], left, base)
    mass = left.cumsum(-1)
    pick = (mass <= s["sample_u"].double()[:, None] * mass[:, -1:]).sum(-1)
    final = torch.where(left > 0, ids, -1).amax(-1)
    pick = torch.minimum(pick, final).to(torch.int32)
    out = torch.cat([torch.where(place < n_acc[:, None], s["tokens"][at] if N else at.int(), -1).int(), pad], dim=-1)
    out = torch.where(torch.arange(D + 1, device=dev) == n_acc[:, None], pick[:, None], out)
    return [out, n_acc.to(torch.int32)]


def _exact_verify(c, seed):
    s = _prepare_verify(c, seed)
    cu, tokens, temps = s["cu"].tolist(), s["tokens"].tolist(), s["temperature"].tolist()
    u, u_last = s["accept_u"].tolist(), s["sample_u"].tolist()
    out = np.full((c["seqs"], c["drafts"] + 1), -1, dtype=np.int32)
    count = np.zeros(c["seqs"], dtype=np.int32)

    def target(r, T):
        x = s["logits"][r].double().cpu().numpy()
        if T == 0:
            p = np.zeros_like(x)
            p[int(np.argmax(x))] = 1.0
            return p
        e = np.exp((x - x.max()) / T)
        return e / e.sum()

    for i in range(c["seqs"]):
        for j in range(cu[i], cu[i + 1] + 1):
            p = target(j + i, temps[i])
            if j < cu[i + 1]:
                q = None if s["probs"] is None else s["probs"][j].double().cpu().numpy()
                if u[j] * (1.0 if q is None else q[tokens[j]]) < p[tokens[j]]:
                    out[i, count[i]] = tokens[j]
                    count[i] += 1
                    continue
                r = p.copy()
                if q is None:
                    r[tokens[j]] = 0.0
                else:
                    r = np.maximum(p - q, 0.0)
                p = r if temps[i] > 0 and r.sum() > 0 else p
            mass = np.cumsum(p)
            k = int(np.searchsorted(mass, u_last[i] * mass[-1], side="right"))
            out[i, count[i]] = min(k, int(np.nonzero(p)[0][-1]))
            break
    return [out, count]


# ---- the interface ----
def prepare(case, seed):
    return {"norm": _prepare_norm, "prefix": _prepare_prefix, "verify": _prepare_verify}[case["call"]](case, seed)


def run(state):
    return {"norm": _run_norm, "prefix": _run_prefix, "verify": _run_verify}[state["case"]["call"]](state)


def exact(case, seed):
    return {"norm": _exact_norm, "prefix": _exact_prefix, "verify": _exact_verify}[case["call"]](case, seed)
