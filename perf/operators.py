"""Cases, plain forms and exact values of the cache operators.

Three operators around the sign-bit / FP8 cache of the forward:

  write    rotary positions on new queries and keys, then the cache's formats: sign
           words of Q, sign words of K and e4m3 codes of V at their slots
  weights  the attention weight every cached key receives from a set of query rows,
           added to a running sum per key
  evict    the keys of each cache row that stay under a budget, by that sum, with the
           first and the newest positions protected, and the move that packs them

Cache rows are (sequence, KV head) pairs; slot t of row r lives in pool row
table[r, t // block] * block + t % block, or r * capacity + t without a table.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False
DEVICE = "cuda"

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FP8 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one sequence decoding far into a long context: latency
        dict(name="write_token", op="write", dtype="bf16", D=128, Hq=32, Hk=8, rot=128, layout="half", seqs=1, tokens=1,
             prompt=False, far=131072, cap=4096, block=16, fused=False),
        # a decode step of a large batch into evicted caches, where the slot is not the position
        dict(name="write_decode", op="write", dtype="f16", D=128, Hq=32, Hk=8, rot=128, layout="half", seqs=256,
             tokens=256, prompt=False, far=32768, cap=1024, block=16, fused=True),
        # ragged prompts of wide heads with rotary positions on a part of each head, 32-bit activations
        dict(name="write_ragged", op="write", dtype="f32", D=256, Hq=16, Hk=4, rot=64, layout="interleaved", seqs=5,
             tokens=1999, prompt=True, far=0, cap=0, block=0, fused=False),
        # whole prompts straight from a fused projection
        dict(name="write_prompt", op="write", dtype="bf16", D=128, Hq=32, Hk=8, rot=128, layout="half", seqs=8,
             tokens=32768, prompt=True, far=0, cap=0, block=16, fused=True),
        # one short sequence: latency
        dict(name="weights_small", op="weights", D=128, Hq=32, Hk=8, seqs=1, ctx_min=333, ctx_max=333, n_q=1, block=16,
             decay=1.0),
        # a decode step of a batch with ragged contexts
        dict(name="weights_decode", op="weights", D=128, Hq=32, Hk=8, seqs=64, ctx_min=2048, ctx_max=8192, n_q=1,
             block=16, decay=1.0),
        # a decode step of one long sequence: few rows, a long axis
        dict(name="weights_long", op="weights", D=128, Hq=32, Hk=8, seqs=1, ctx_min=131072, ctx_max=131072, n_q=1,
             block=128, decay=0.99),
        # the last queries of prompts, before their caches are cut to a budget
        dict(name="weights_window", op="weights", D=128, Hq=32, Hk=8, seqs=4, ctx_min=8000, ctx_max=16384, n_q=64,
             block=16, decay=1.0),
        # one key over the budget in every row, as in each decode step at the budget
        dict(name="evict_step", op="evict", D=128, rows=512, ctx_min=4097, ctx_max=4097, keep=4096, per_row=False, sink=4,
             recent=64, block=16, slot_scale=False),
        # budgets of their own for each row, wide heads, a scale per slot, contiguous rows
        dict(name="evict_odd", op="evict", D=256, rows=24, ctx_min=700, ctx_max=2111, keep=501, per_row=True, sink=0,
             recent=33, block=0, slot_scale=True),
        # few rows of a long cache
        dict(name="evict_long", op="evict", D=128, rows=8, ctx_min=120001, ctx_max=131072, keep=16384, per_row=False,
             sink=4, recent=256, block=64, slot_scale=False),
        # prompts cut to a budget
        dict(name="evict_prompt", op="evict", D=128, rows=128, ctx_min=16384, ctx_max=32768, keep=4096, per_row=False,
             sink=4, recent=64, block=16, slot_scale=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["write", "weights", "evict"])
    D = rng.choice([128, 128, 256])
    Hk = rng.choice([1, 2, 4, 8])
    Hq = Hk * rng.choice([1, 2, 4, 8])
    if Hq > 32:
        Hq = 32
    block = rng.choice([0, 8, 16, 20, 64, 128])
    if op == "write":
        rot = 2 * rng.randint(1, D // 2) if rng.random() < 0.3 else rng.choice([D, D // 2, D // 4])
        dtype = rng.choice(["bf16", "f16", "f32"])
        prompt = rng.random() < 0.5
        most = 32768 * 128 // D // (2 if dtype == "f32" else 1)
        tokens = _log(rng, 1, most) if prompt else _log(rng, 1, 512)
        seqs = min(tokens, rng.randint(1, 16)) if prompt else tokens
        return dict(op=op, dtype=dtype, D=D, Hq=Hq, Hk=Hk, rot=rot, layout=rng.choice(["half", "interleaved"]), seqs=seqs,
                    tokens=tokens, prompt=prompt, far=0 if prompt else _log(rng, 64, 131072),
                    cap=0 if prompt else _log(rng, 17, 2048), block=block, fused=rng.random() < 0.5)
    if op == "weights":
        n_q = rng.choice([1, 1, 1, _log(rng, 2, 64)])
        ctx = _log(rng, 1, 131072)
        # no more (query, key) products than the widest listed case, no more keys than the longest
        most = 4 * 8 * 16384 * 64 * 4 * 128 // (ctx * n_q * Hq * D)
        seqs = _log(rng, 1, max(1, min(64, most, 4194304 // (ctx * Hk))))
        if ctx * n_q * Hq * D * seqs > 4 * 8 * 16384 * 64 * 4 * 128:
            n_q = 1
        return dict(op=op, D=D, Hq=Hq, Hk=Hk, seqs=seqs, ctx_min=max(1, ctx // rng.choice([1, 2, 8])), ctx_max=ctx, n_q=n_q,
                    block=block, decay=rng.choice([1.0, 0.95]))
    ctx = _log(rng, 2, 131072)
    rows = _log(rng, 1, max(1, min(512, 4194304 * 128 // D // ctx)))
    keep = max(1, ctx - 1) if rng.random() < 0.4 else _log(rng, 1, ctx)
    recent = rng.randint(0, min(keep, 100) // 2)
    return dict(op=op, D=D, rows=rows, ctx_min=max(1, ctx // rng.choice([1, 2, 8])), ctx_max=ctx, keep=keep,
                per_row=rng.random() < 0.3, sink=min(4, keep - recent), recent=recent, block=block,
                slot_scale=rng.random() < 0.3)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _lengths(seed, n, lo, hi):
    """n lengths in [lo, hi], the longest among them."""
    r = random.Random(seed * 7919 + n)
    lens = [r.randint(lo, hi) for _ in range(n)]
    lens[r.randrange(n)] = hi
    return lens


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _pages(g, rows, cap, block):
    """(table or None, block, pages a row, pool rows): every row's pages lie anywhere in the pool."""
    if block == 0:
        return None, cap, 1, rows * cap
    nb = -(-cap // block)
    table = torch.randperm(rows * nb, generator=g, device=DEVICE).to(torch.int32).view(rows, nb)
    return table, block, nb, rows * nb * block


def _codes(g, rows, D):
    return torch.randn(rows, D, generator=g, device=DEVICE, dtype=torch.float16).mul_(100).clamp_(-448, 448).to(FP8).view(torch.uint8)


def _words(g, rows, D):
    return torch.randint(-2**31, 2**31, (rows, D // 32), generator=g, device=DEVICE, dtype=torch.int64).to(torch.int32)


def _table(n, rot):
    """cos and sin of position * 10000^(-2i/rot): angles in 64 bits, each value rounded once."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE) / rot)
    angle = torch.arange(n, dtype=torch.float64, device=DEVICE)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], dim=1).float()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"write": _prepare_write, "weights": _prepare_weights, "evict": _prepare_evict}[case["op"]](case, seed, g)


def _prepare_write(c, seed, g):
    D, Hq, Hk, T, B = c["D"], c["Hq"], c["Hk"], c["tokens"], c["seqs"]
    dt = DTYPES[c["dtype"]]
    slots = None
    if c["prompt"]:
        # the case has its lengths, the seed their order: shapes do not depend on it
        cuts = sorted(random.Random(T * 31 + B).sample(range(1, T), B - 1))
        lens = [b - a for a, b in zip([0] + cuts, cuts + [T])]
        random.Random(seed).shuffle(lens)
        cap = seq_q = max(lens)
        seq = torch.repeat_interleave(torch.arange(B, device=DEVICE), torch.tensor(lens, device=DEVICE)).to(torch.int32)
        pos = torch.cat([torch.arange(n, device=DEVICE) for n in lens]).to(torch.int32)
        far = cap
    else:
        cap, seq_q, far = c["cap"], 1, c["far"]
        seq = torch.randperm(T, generator=g, device=DEVICE).to(torch.int32)
        pos = torch.randint(far // 2, far, (T,), generator=g, device=DEVICE).to(torch.int32)
        slots = torch.randint(0, cap, (T, Hk), generator=g, device=DEVICE).to(torch.int32)
    if c["fused"]:
        x = torch.randn(T, Hq + 2 * Hk, D, generator=g, device=DEVICE, dtype=dt)
        q, k, v = x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]
    else:
        q, k, v = (torch.randn(T, h, D, generator=g, device=DEVICE, dtype=dt) for h in (Hq, Hk, Hk))
    table, block, nb, pool = _pages(g, B * Hk, cap, c["block"])
    scale = (torch.rand(Hk, generator=g, device=DEVICE) + 0.5) * (4.0 / 448.0)
    return dict(op="write", q=q, k=k, v=v, seq=seq, pos=pos, slots=slots, rope=_table(far, c["rot"]), rot=c["rot"],
                layout=c["layout"], table=table, block=block, nb=nb, scale=scale, seq_q=seq_q,
                q_words=torch.zeros(B * Hq * seq_q, D // 32, dtype=torch.int32, device=DEVICE), k_cache=_words(g, pool, D),
                v_cache=_codes(g, pool, D), slot_pos=torch.full((B * Hk, nb * block), -1, dtype=torch.int32, device=DEVICE))


def _prepare_weights(c, seed, g):
    D, Hk, n_q = c["D"], c["Hk"], c["n_q"]
    lens = _lengths(seed, c["seqs"], c["ctx_min"], c["ctx_max"])
    rows, cap = c["seqs"] * Hk, c["ctx_max"]
    table, block, nb, pool = _pages(g, rows, cap, c["block"])
    ctx = _ints(lens).repeat_interleave(Hk)
    seq_q = 1 if n_q == 1 else cap
    w = torch.rand(rows, nb * block, generator=g, device=DEVICE)
    return dict(op="weights", q=_words(g, rows * (c["Hq"] // Hk) * seq_q, D), k_cache=_words(g, pool, D), ctx=ctx, table=table,
                block=block, nb=nb, weights=w, out=torch.zeros_like(w), seq_q=seq_q, D=D, group=c["Hq"] // Hk, n_q=n_q,
                first=None if n_q == 1 else ctx - n_q, causal=n_q > 1, decay=c["decay"], inv=1.0 / math.sqrt(D))


def _prepare_evict(c, seed, g):
    D, rows, cap = c["D"], c["rows"], c["ctx_max"]
    ctx = _ints(_lengths(seed, rows, c["ctx_min"], cap))
    table, block, nb, pool = _pages(g, rows, cap, c["block"])
    ld = nb * block
    # weights sums are heavy-tailed, and keys that nothing has looked at yet share the value 0
    w = torch.randn(rows, ld, generator=g, device=DEVICE).abs_().pow_(4)
    w.masked_fill_(torch.rand(rows, ld, generator=g, device=DEVICE) < 0.05, 0.0)
    # earlier moves have left the positions out of order and with gaps; the newest keys come last
    order = torch.rand(rows, ld, generator=g, device=DEVICE)
    at = torch.arange(ld, device=DEVICE)[None, :]
    order = torch.where(at >= (ctx[:, None] - c["recent"]), 2.0 + at, order.double())
    pos = (order.argsort(dim=1).argsort(dim=1) * 2).to(torch.int32)
    keep = c["keep"]
    if c["per_row"]:
        keep = _ints(_lengths(seed + 1, rows, max(1, keep // 2), keep))
    return dict(op="evict", k_cache=_words(g, pool, D), v_cache=_codes(g, pool, D), ctx=ctx, table=table, block=block, nb=nb,
                weights=w, pos=pos, keep=keep, sink=c["sink"], recent=c["recent"],
                scale=torch.rand(pool, generator=g, device=DEVICE) if c["slot_scale"] else None,
                ctx_out=torch.zeros_like(ctx), w_out=torch.zeros_like(w), pos_out=torch.full_like(pos, -1))


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _framework():
    path = os.path.join(os.getcwd(), "hyperion-fa3-kernel-_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import hyperion_b200

    return hyperion_b200


def run(s):
    if own:
        return _run_own(s)
    return {"write": _plain_write, "weights": _plain_weights, "evict": _plain_evict}[s["op"]](s)


def _run_own(s):
    h = _framework()
    if s["op"] == "write":
        h.rope_cache_write(s["q"], s["k"], s["v"], s["seq"], s["pos"], s["rope"], s["table"], s["block"], s["nb"], s["scale"],
                           s["q_words"], s["k_cache"], s["v_cache"], layout=s["layout"], seq_q=s["seq_q"], slots=s["slots"],
                           slot_positions=s["slot_pos"])
        return _outputs_write(s)
    if s["op"] == "weights":
        h.accumulate_key_weights(s["q"], s["k_cache"], s["ctx"], s["table"], s["weights"], s["seq_q"], s["D"], s["block"],
                                 s["nb"], s["inv"], s["causal"], kv_group=s["group"], q_first=s["first"], n_q=s["n_q"],
                                 decay=s["decay"], out=s["out"])
        return [s["out"]]
    h.evict_keys(s["k_cache"], s["v_cache"], s["ctx"], s["table"], s["block"], s["nb"], s["weights"], s["pos"], s["keep"],
                 sink=s["sink"], recent=s["recent"], V_scale=s["scale"], context_lens_out=s["ctx_out"],
                 weights_out=s["w_out"], positions_out=s["pos_out"])
    return _outputs_evict(s)


def _outputs_write(s):
    return [s["q_words"], s["k_cache"], s["v_cache"].view(FP8), s["slot_pos"]]


def _outputs_evict(s):
    return [s["ctx_out"], s["w_out"], s["pos_out"], s["k_cache"], s["v_cache"].view(FP8)] + ([] if s["scale"] is None else [s["scale"]])


def _pool_rows(s, rows, slots):
    """Pool rows of the given slots of the given cache rows."""
    if s["table"] is None:
        return rows * s["block"] + slots
    return s["table"][rows, slots // s["block"]].long() * s["block"] + slots % s["block"]


def _sign_words(x):
    bits = (x >= 0).view(*x.shape[:-1], x.shape[-1] // 32, 32).long()
    words = (bits << torch.arange(32, device=x.device)).sum(-1)
    return (words - ((words >> 31) << 32)).to(torch.int32)


def _plain_write(s):
    seq, pos = s["seq"].long(), s["pos"].long()
    T, Hq, D = s["q"].shape
    Hk, rot = s["k"].shape[1], s["rot"]
    # the sign of a sum next to zero needs more than 32 bits: products of two 32-bit values are exact in 64
    cos, sin = s["rope"][pos].double()[:, None].unbind(2)

    def rotated(x):
        x = x.double()
        if s["layout"] == "half":
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], dim=-1)
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), x[..., rot:]], dim=-1)

    q_idx = pos if s["seq_q"] > 1 else torch.zeros_like(pos)
    s["q_words"][((seq[:, None] * Hq + torch.arange(Hq, device=seq.device)) * s["seq_q"] + q_idx[:, None])] = _sign_words(rotated(s["q"]))
    rows = seq[:, None] * Hk + torch.arange(Hk, device=seq.device)
    slots = (pos[:, None].expand(T, Hk) if s["slots"] is None else s["slots"]).long()
    at = _pool_rows(s, rows, slots)
    s["k_cache"][at] = _sign_words(rotated(s["k"]))
    s["v_cache"][at] = (s["v"].float() / s["scale"][:, None]).clamp(-448, 448).to(FP8).view(torch.uint8)
    s["slot_pos"][rows, slots] = s["pos"][:, None].expand(T, Hk)
    return _outputs_write(s)


def _signs(words):
    """+1 / -1 for each bit of the words' rows."""
    bits = (words[..., None] >> torch.arange(32, dtype=torch.int32, device=words.device)) & 1
    return bits.flatten(-2).float().mul_(2).sub_(1)


def _plain_weights(s):
    n, g, n_q, cap = s["ctx"].numel(), s["group"], s["n_q"], s["nb"] * s["block"]
    dev = s["ctx"].device
    rows, at = torch.arange(n, device=dev)[:, None], torch.arange(cap, device=dev)[None, :]
    ctx = s["ctx"].long()[:, None]
    first = torch.zeros_like(ctx) if s["first"] is None else s["first"].long()[:, None]
    q_idx = (first + torch.arange(n_q, device=dev))[:, None, :].expand(n, g, n_q)
    real = (q_idx >= 0) & (q_idx < s["seq_q"])
    q = s["q"].view(n, g, s["seq_q"], -1)[rows[:, :, None], torch.arange(g, device=dev)[None, :, None], q_idx.clamp(0, s["seq_q"] - 1)]
    keys = _signs(s["k_cache"][_pool_rows(s, rows, at)])
    x = torch.matmul(_signs(q).flatten(1, 2), keys.transpose(1, 2)) * s["inv"]  # [n, g * n_q, cap]
    del keys
    seen = (at[:, None] < ctx[:, None]) & real.reshape(n, -1, 1)
    if s["causal"]:
        seen = seen & (at[:, None] <= q_idx.reshape(n, -1, 1))
    x = x.masked_fill_(~seen, -math.inf)
    p = (x - x.amax(-1, keepdim=True).clamp_min(-1e30)).clamp_min_(-80.0).exp_().masked_fill_(~seen, 0.0)
    del x
    total = (p / p.sum(-1, keepdim=True).clamp_min(1e-30)).sum(1)
    s["out"].copy_(torch.where(at < ctx, s["decay"] * s["weights"] + total, s["out"]))
    return [s["out"]]


def _plain_evict(s):
    w, pos, ctx = s["weights"], s["pos"].long(), s["ctx"].long()[:, None]
    at = torch.arange(w.shape[1], device=w.device)[None, :]
    valid = at < ctx
    keep = s["keep"].long()[:, None] if torch.is_tensor(s["keep"]) else torch.full_like(ctx, s["keep"])
    new = torch.minimum(ctx, keep)
    newest = pos.masked_fill(~valid, -1).amax(1, keepdim=True)
    protected = (pos < s["sink"]) | (pos > newest - s["recent"])
    # an order of whole numbers: protected keys first, then by weight (NaN last), equal ones by slot
    bits = (w + 0.0).view(torch.int32).long()
    rank = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits).masked_fill(torch.isnan(w), -2**31)
    rank = torch.where(protected, 2**32, rank).masked_fill(~valid, -2**40)
    order = rank.argsort(dim=1, descending=True, stable=True)
    kept = torch.zeros_like(valid).scatter_(1, order, at < new)
    # the i-th slot under the budget that empties takes the i-th kept key beyond it
    row, dst = (~kept & (at < new)).nonzero(as_tuple=True)
    _, src = (kept & (at >= new)).nonzero(as_tuple=True)
    to, frm = _pool_rows(s, row, dst), _pool_rows(s, row, src)
    s["k_cache"][to] = s["k_cache"][frm]
    s["v_cache"][to] = s["v_cache"][frm]
    if s["scale"] is not None:
        s["scale"][to] = s["scale"][frm]
    w_new, p_new = w.clone(), s["pos"].clone()
    w_new[row, dst], p_new[row, dst] = w[row, src], s["pos"][row, src]
    s["w_out"].copy_(torch.where(at < new, w_new, torch.where(valid, 0.0, s["w_out"])))
    s["pos_out"].copy_(torch.where(at < new, p_new, torch.where(valid, -1, s["pos_out"])))
    s["ctx_out"].copy_(new[:, 0])
    return _outputs_evict(s)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(c):
    D = c["D"]
    if c["op"] == "write":
        size = 4 if c["dtype"] == "f32" else 2
        T, Hq, Hk = c["tokens"], c["Hq"], c["Hk"]
        # activations and cos / sin rows in; sign words, codes and slot positions out
        distinct = T if not c["prompt"] else -(-T // c["seqs"])
        return dict(bytes=T * (Hq + 2 * Hk) * D * size + distinct * c["rot"] * 4 + T * 8 + T * Hq * D // 8 + T * Hk * (D // 8 + D + 4),
                    flops=T * (Hq + Hk) * c["rot"] * 3 + T * Hk * D)
    if c["op"] == "weights":
        keys = c["seqs"] * c["Hk"] * (c["ctx_min"] + c["ctx_max"]) // 2
        pairs = keys * c["n_q"] * (c["Hq"] // c["Hk"])
        # key words and sums in, sums out, query words; a product and a softmax step per pair
        return dict(bytes=keys * (D // 8 + 8) + c["seqs"] * c["Hq"] * c["n_q"] * D // 8, flops=pairs * (2 * D + 4))
    keys = c["rows"] * (c["ctx_min"] + c["ctx_max"]) // 2
    n, k = max(1, (c["ctx_min"] + c["ctx_max"]) // 2), min(c["keep"], (c["ctx_min"] + c["ctx_max"]) // 2)
    fixed = min(k, c["recent"])
    moved = c["rows"] * min(n - k, fixed + (k - fixed) * max(0, n - k - fixed) // n)
    # sums and positions in and out; each moved key read and written once
    return dict(bytes=keys * 16 + moved * 2 * (D // 8 + D + (4 if c["slot_scale"] else 0)), flops=keys * 4)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    return {"write": _exact_write, "weights": _exact_weights, "evict": _exact_evict}[c["op"]](s)


def _exact_write(s):
    T, Hq, D = s["q"].shape
    Hk, rot = s["k"].shape[1], s["rot"]
    d = np.arange(D)
    if s["layout"] == "half":
        pair, second = d % max(1, rot // 2), d >= rot // 2
        other = np.where(second, d - rot // 2, d + rot // 2)
    else:
        pair, second, other = d // 2, d % 2 == 1, d ^ 1
    turned = d < rot
    pair, other = np.where(turned, pair, 0), np.where(turned, other, d)
    rows = s["rope"].double()[s["pos"].long()]
    on = torch.tensor(turned, device=DEVICE)
    c = torch.where(on, rows[:, 0][:, pair], 1.0)[:, None]
    sn = torch.where(on, rows[:, 1][:, pair] * torch.tensor(np.where(second, 1.0, -1.0), device=DEVICE), 0.0)[:, None]
    weight = 2.0 ** torch.arange(32, dtype=torch.float64, device=DEVICE)

    def words(x):
        x = x.double()
        up = (x * c + x[..., other] * sn >= 0).double().view(x.shape[0], x.shape[1], D // 32, 32)
        v = (up * weight).sum(-1)
        return torch.where(v >= 2.0**31, v - 2.0**32, v).to(torch.int32)

    qw, kw = words(s["q"]), words(s["k"])
    value = s["v"].double() / s["scale"].double()[:, None]
    q_out, k_out, p_out = s["q_words"].clone(), s["k_cache"].clone(), s["slot_pos"].clone()
    v_out = s["v_cache"].view(FP8).double()
    seq, pos = s["seq"].long(), s["pos"].long()
    for h in range(Hq):
        q_out[(seq * Hq + h) * s["seq_q"] + (pos if s["seq_q"] > 1 else 0)] = qw[:, h]
    for h in range(Hk):
        slot = pos if s["slots"] is None else s["slots"][:, h].long()
        row = seq * Hk + h
        page = row * s["nb"] + slot // s["block"]
        page = page if s["table"] is None else s["table"].view(-1).long()[page]
        at = page * s["block"] + slot % s["block"]
        k_out[at], v_out[at] = kw[:, h], value[:, h].clamp(-448.0, 448.0)
        p_out[row, slot] = s["pos"]
    return [q_out, k_out, v_out, p_out]


def _exact_weights(s):
    g, n_q, W = s["group"], s["n_q"], s["D"] // 32
    q = s["q"].view(-1, g, s["seq_q"], W).long() & 0xFFFFFFFF
    out = s["out"].double()
    first = [0] * s["ctx"].numel() if s["first"] is None else s["first"].tolist()
    for r, n in enumerate(s["ctx"].tolist()):
        t = torch.arange(n, device=DEVICE)
        at = r * s["block"] * s["nb"] + t if s["table"] is None else s["table"][r].long()[t // s["block"]] * s["block"] + t % s["block"]
        lo, hi = max(0, first[r]), min(s["seq_q"], first[r] + n_q)
        x = (q[r, :, lo:hi].reshape(-1, 1, W)) ^ (s["k_cache"][at].long() & 0xFFFFFFFF)
        # bits counted in fields of 2, 4, 8 and then all at once
        x = x - ((x >> 1) & 0x55555555)
        x = (x & 0x33333333) + ((x >> 2) & 0x33333333)
        x = (((x + (x >> 4)) & 0x0F0F0F0F) * 0x01010101 >> 24) & 0xFF
        x = (s["D"] - 2 * x.sum(-1)).double() * s["inv"]
        if s["causal"]:
            x[t[None, :] > torch.arange(lo, hi, device=DEVICE).repeat(g)[:, None]] = -math.inf
        e = torch.exp(x - x.max(1, keepdim=True).values)  # |x| stays far from the clamp at -80
        out[r, :n] = s["decay"] * s["weights"][r, :n].double() + (e / e.sum(1, keepdim=True)).sum(0)
    return [out]


def _exact_evict(s):
    w, pos = s["weights"].cpu().numpy(), s["pos"].cpu().numpy()
    w_out, p_out = s["w_out"].cpu().numpy().astype(np.float64), s["pos_out"].cpu().numpy()
    lens, ends, moves = s["ctx"].tolist(), [], []
    for r, n in enumerate(lens):
        keep = min(n, int(s["keep"][r]) if torch.is_tensor(s["keep"]) else s["keep"])
        p, x = pos[r, :n], w[r, :n]
        guard = (p < s["sink"]) | (p > p.max() - s["recent"])
        stay = np.zeros(n, bool)
        stay[np.lexsort((np.arange(n), np.where(guard, 0.0, -x), ~guard))[:keep]] = True
        empty, late = np.flatnonzero(~stay[:keep]), keep + np.flatnonzero(stay[keep:])
        frm = np.arange(keep)
        frm[empty] = late
        w_out[r, :keep], p_out[r, :keep] = x[frm], p[frm]
        w_out[r, keep:n], p_out[r, keep:n] = 0.0, -1
        ends.append(keep)
        moves.append(np.stack([np.full(empty.size, r), empty, late]))
    row, dst, src = (torch.tensor(np.concatenate(x), device=DEVICE) for x in zip(*moves))

    def place(t):
        page = row * s["nb"] + t // s["block"]
        return (page if s["table"] is None else s["table"].view(-1).long()[page]) * s["block"] + t % s["block"]

    k, v = s["k_cache"].clone(), s["v_cache"].view(FP8).double()
    k[place(dst)], v[place(dst)] = s["k_cache"][place(src)], v[place(src)]
    out = [_ints(ends), torch.tensor(w_out, device=DEVICE), torch.tensor(p_out, device=DEVICE), k, v]
    if s["scale"] is not None:
        scale = s["scale"].double()
        scale[place(dst)] = scale[place(src)]
        out.append(scale)
    return out
