"""Cases of the paged-cache operators: the attention half of a trunk layer.

Each case is one call of ``soraku_amd.ops`` on a cache in pages:

* ``append``  per-head norm and rotation of new tokens' q and k, k and v into
              their pages (``ops.paged_append``);
* ``attend``  attention of the new tokens over the pages, with or without a
              sliding window and first tokens that stay visible
              (``ops.paged_attention``);
* ``mass``    the attention weight every cached key got, added to its account
              (``ops.paged_attention_mass``);
* ``evict``   the keys with the largest accounts moved to fresh pages
              (``ops.paged_evict``).

``own`` chooses between those calls and the plain form: gathered pages and
elementary torch operations in 32 bits (angles in 64), rounded once at the end.

A case has ``seqs`` sequences of up to ``new`` new tokens each, whose caches
hold up to ``ctx`` tokens with the new ones; several sequences are ragged, from
half to all of those.  Head layouts are the package's trunk shapes (16 query and
8 key heads of 128) and, drawn, others from one key head to as many as query
heads and down to the tiny shape's heads of 16.  Pages lie in the pool in random
order.  Norm gains and rotations leave scores of a spread of about two, so some
keys matter far more than others.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
EPS = 1e-6           # the trunk's norm
THETA = 1e6          # the trunk's rotation base
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "soraku-tts_amd")
_OPS = []


def _ops():
    """``soraku_amd.ops``, imported when its calls are first wanted."""
    if not _OPS:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        from soraku_amd import ops
        _OPS.append(ops)
    return _OPS[0]


# ------------------------------------------------------------------ cases

def _case(kind, seqs, new, ctx, *, hq=16, hkv=8, hd=128, page=64, q_bf16=False, kv_bf16=True, window=0, sinks=0,
          keep=0, recent=0, mass=False):
    return dict(kind=kind, seqs=seqs, new=new, ctx=ctx, hq=hq, hkv=hkv, hd=hd, page=page, q_bf16=q_bf16,
                kv_bf16=kv_bf16, window=window, sinks=sinks, keep=keep, recent=recent, mass=mass)


def listed():
    return [
        # one frame of 16 utterances with CFG: 32 tokens, all latency
        dict(_case("append", 32, 1, 657, page=16), name="append_step_32rows"),
        # a serving batch's ragged voice-cloning prefixes, 16 utterances with CFG, accounts kept
        dict(_case("append", 32, 240, 240, mass=True), name="append_prompts_32rows"),
        # one utterance with CFG, FP32: one token each at the end of a 240-frame utterance
        dict(_case("attend", 2, 1, 481, kv_bf16=False), name="attend_pair_f32"),
        # the throughput batch's frame: 32 ragged rows, BF16 cache in small pages
        dict(_case("attend", 32, 1, 657, page=16), name="attend_step_32rows"),
        # hour-long speech: single tokens of a CFG pair over a very long cache
        dict(_case("attend", 2, 1, 61441), name="attend_step_long"),
        # the prefix of a CFG pair, FP32 throughout
        dict(_case("attend", 2, 387, 387, kv_bf16=False), name="attend_prompt_pair_f32"),
        # a long text's chunk over what came before it, everything BF16
        dict(_case("attend", 1, 2047, 16384, q_bf16=True), name="attend_chunk_bf16"),
        # chunks of four streams that see a window and the first tokens (text, speaker)
        dict(_case("attend", 4, 1500, 9001, window=1024, sinks=96), name="attend_window_chunk"),
        # accounts of a frame of 16 long utterances with CFG
        dict(_case("mass", 32, 1, 4800), name="mass_step_32rows"),
        # accounts of a prompt's own tokens
        dict(_case("mass", 2, 1800, 3600), name="mass_prompt_pair"),
        # long utterances cut back to a budget between frames
        dict(_case("evict", 32, 1, 4800, sinks=96, recent=256, keep=2400), name="evict_32rows"),
        # one pair's very long cache, FP32, cut to an eighth
        dict(_case("evict", 2, 1, 61440, kv_bf16=False, sinks=16, recent=1024, keep=7680), name="evict_long_f32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "mass", "evict"])
    top = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        hq, hkv, hd = rng.choice([(16, 8, 128)] * 6 + [(16, 16, 128), (16, 4, 128), (12, 4, 64), (8, 1, 64), (6, 3, 32),
                                                       (4, 2, 16)])
        q_bf16, kv_bf16 = rng.choice([(False, False), (False, True), (False, True), (True, True)])
        c = _case(kind, rng.choice([1, 2, _log_int(rng, 1, 32)]), 1, 1, hq=hq, hkv=hkv, hd=hd,
                  page=rng.choice([16, 32, 48, 64, 128, 256]), q_bf16=q_bf16, kv_bf16=kv_bf16)
        c["ctx"] = _log_int(rng, 1, 61441)
        if kind != "evict" and rng.random() < 0.6:
            c["new"] = min(c["ctx"], _log_int(rng, 2, 2047))
        if kind in ("attend", "mass") and rng.random() < 0.35:
            c["window"], c["sinks"] = _log_int(rng, 1, 4096), rng.choice([0, 4, _log_int(rng, 1, 256)])
        if kind == "append":
            c["mass"] = rng.random() < 0.5
        if kind == "evict":
            c["keep"] = _log_int(rng, 1, max(1, c["ctx"]))
            c["sinks"] = rng.choice([0, min(4, c["keep"]), rng.randint(0, min(256, c["keep"]))])
            c["recent"] = rng.randint(0, c["keep"] - c["sinks"])
        if _cost(c) <= top and _plain_bytes(c) <= 2.5e10 and _pool_bytes(c) <= 2.5e9:
            return c


def _plain_bytes(case):
    """What the plain form holds at once, roughly: scores and gathered pages."""
    pairs = case["seqs"] * case["new"] * case["hq"] * case["ctx"] if case["kind"] in ("attend", "mass") else 0
    return 4 * (4 * pairs + 8 * case["seqs"] * case["hkv"] * case["hd"] * case["ctx"])


def _pool_bytes(case):
    return case["seqs"] * (case["ctx"] + case["keep"]) * case["hkv"] * case["hd"] * (4 if case["kv_bf16"] else 8)


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / (1.4e14 if not case["kv_bf16"] else 1.2e15 if case["q_bf16"] else 4e14)


def _lens(case):
    """(new tokens, cache length with them) of each sequence."""
    n, out = case["seqs"], []
    for u in range(n):
        f = 1.0 if n == 1 else 0.5 + 0.5 * ((7 * u) % n) / (n - 1)
        new = max(1, round(case["new"] * f))
        out.append((new, max(new, round(case["ctx"] * f))))
    return out


def _visible(case, new, length):
    """(query, key) pairs of one sequence for one query head, and the keys that any query sees."""
    p = np.arange(length - new, length, dtype=np.int64)
    if not case["window"]:
        return int((p + 1).sum()), length
    lo = np.maximum(0, p + 1 - case["window"])
    return int((p + 1 - lo + np.minimum(lo, case["sinks"])).sum()), int(length - lo[0] + min(lo[0], case["sinks"]))


def work(case):
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    qb, kb = 2 if case["q_bf16"] else 4, 2 if case["kv_bf16"] else 4
    rows = _lens(case)
    t = sum(n for n, _ in rows)
    if case["kind"] == "append":
        return {"bytes": t * ((2 * hq + 2 * hkv) * hd * qb + 2 * hkv * hd * kb + (4 * hkv if case["mass"] else 0)),
                "flops": 10 * t * (hq + hkv) * hd}
    if case["kind"] == "evict":
        kept = sum(min(case["keep"], n) for _, n in rows)
        return {"bytes": hkv * (4 * sum(n for _, n in rows) + kept * (4 * hd * kb + 8)), "flops": 0}
    see = [_visible(case, *r) for r in rows]
    pairs, keys = hq * sum(s[0] for s in see), hkv * sum(s[1] for s in see)
    if case["kind"] == "attend":
        return {"bytes": 2 * t * hq * hd * qb + 2 * keys * hd * kb, "flops": 4 * hd * pairs}
    return {"bytes": t * hq * (hd * qb + 4) + keys * (hd * kb + 8), "flops": 2 * hd * pairs}


# ------------------------------------------------------------------ inputs

def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 29)
    rng = np.random.default_rng([int(seed), 11])
    hq, hkv, hd, page, n = case["hq"], case["hkv"], case["hd"], case["page"], case["seqs"]
    qt = torch.bfloat16 if case["q_bf16"] else torch.float32
    kt = torch.bfloat16 if case["kv_bf16"] else torch.float32
    rows = _lens(case)
    new, lens = np.array([r[0] for r in rows]), np.array([r[1] for r in rows])
    width = -(-int(lens.max()) // page)
    dst_width = -(-case["keep"] // page)
    n_pages = n * (width + dst_width)
    order = rng.permutation(n_pages)
    starts = np.concatenate(([0], np.cumsum(new)))
    t = int(starts[-1])
    at = np.arange(t)
    seq = np.repeat(np.arange(n), new)

    def rand(*shape, scale=1.0, dtype=torch.float32):
        x = torch.randn(*shape, generator=g, device=DEV, dtype=dtype)
        return x if scale == 1.0 else x.mul_(scale)

    s = dict(case=case, table=_i32(order[: n * width].reshape(n, width)), lens=_i32(lens), starts=_i32(starts),
             most_new=int(new.max()), tokens=t, seq=torch.from_numpy(seq).to(DEV),
             slot=torch.from_numpy(lens[seq] - new[seq] + at - starts[seq]).to(DEV),
             index=torch.from_numpy(at - starts[seq]).to(DEV), scale=hd ** -0.5)
    if case["kind"] != "mass":
        s["v"] = rand(n_pages, hkv, page, hd, dtype=kt)
    s["k"] = rand(n_pages, hkv, page, hd, scale=1.4, dtype=kt)
    if case["kind"] == "append":
        s["qkv"] = rand(t, (hq + 2 * hkv) * hd, scale=0.7, dtype=qt)
        s["q_gain"], s["k_gain"] = rand(hd, scale=0.1).add_(1.2), rand(hd, scale=0.1).add_(1.2)
        s["inv_freq"] = torch.from_numpy((THETA ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)).to(DEV)
        # positions run on where a cache was cut back earlier, so they can be past the slots
        s["positions"] = _i32(lens[seq] - new[seq] + at - starts[seq] + rng.integers(0, 100000, n)[seq])
        s["mass"] = rand(n_pages, hkv, page).abs_() if case["mass"] else None
    else:
        s["q"] = rand(t, hq, hd, scale=1.4, dtype=qt)
    if case["kind"] in ("mass", "evict"):
        # accounts as attention leaves them: a few large ones, many near nothing, some exactly nothing
        m = rand(n_pages, hkv, page).mul_(2.0).exp_().mul_(0.01)
        s["mass"] = m.mul_((torch.rand(n_pages, hkv, page, generator=g, device=DEV) > 0.05).float())
    if case["kind"] == "mass":
        # the softmax statistics that the attention before it left
        s["lse"] = _plain_scores(s)[1][s["seq"], s["index"]].contiguous()
    if case["kind"] == "evict":
        s["dst"] = _i32(order[n * width:].reshape(n, dst_width))
    return s


# ------------------------------------------------------------------ plain form

def _gathered(pages, table, length):
    """[seqs, heads, length, ...] of a page pool, in 32 bits."""
    x = pages[table.long()].transpose(1, 2).float()
    return x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:])[:, :, :length]


def _plain_scores(s):
    """Masked scores [seqs, key heads, group, new, keys] and lse [seqs, new, query heads]."""
    c = s["case"]
    n, hkv, gr, hd, length = c["seqs"], c["hkv"], c["hq"] // c["hkv"], c["hd"], int(s["table"].shape[1]) * c["page"]
    q = torch.zeros(n, s["most_new"], c["hq"], hd, device=DEV)
    q[s["seq"], s["index"]] = s["q"].float()
    q = q.view(n, -1, hkv, gr, hd).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, hd)
    k = _gathered(s["k"], s["table"], length)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n, hkv, gr, -1, length).mul_(s["scale"])
    new = s["starts"].diff().long()
    p = (s["lens"].long() - new)[:, None] + torch.arange(s["most_new"], device=DEV)
    j = torch.arange(length, device=DEV)
    see = (j <= p[:, :, None]) & (torch.arange(s["most_new"], device=DEV) < new[:, None])[:, :, None]
    if c["window"]:
        see &= (j > p[:, :, None] - c["window"]) | (j < c["sinks"])
    x = x.masked_fill_(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min_(-3e38)
    total = (x - top).exp_().sum(-1, keepdim=True)
    lse = (top + total.log()).squeeze(-1)
    return x, lse.permute(0, 3, 1, 2).reshape(n, -1, c["hq"])


def _plain_attend(s):
    c = s["case"]
    x, lse = _plain_scores(s)
    n, hkv, gr, m, length = x.shape
    top = lse.view(n, m, hkv, gr).permute(0, 2, 3, 1)[..., None].clamp_min(-3e38)
    p = x.sub_(top).exp_()
    o = torch.matmul(p.view(n, hkv, gr * m, length), _gathered(s["v"], s["table"], length))
    o = o.view(n, hkv, gr, m, c["hd"]).permute(0, 3, 1, 2, 4).reshape(n, m, c["hq"], c["hd"])
    return o[s["seq"], s["index"]].to(s["q"].dtype), lse[s["seq"], s["index"]]


def _plain_mass(s):
    c = s["case"]
    x, lse = _plain_scores(s)
    n, hkv, gr, m, length = x.shape
    top = torch.zeros(n, m, c["hq"], device=DEV)
    top[s["seq"], s["index"]] = s["lse"]
    p = x.sub_(top.view(n, m, hkv, gr).permute(0, 2, 3, 1)[..., None]).exp_()
    add = p.sum((2, 3)).view(n, hkv, -1, c["page"]).transpose(1, 2)
    s["mass"][s["table"].long()] += add
    return s["mass"]


def _plain_append(s):
    c = s["case"]
    hq, hkv, hd, page = c["hq"], c["hkv"], c["hd"], c["page"]
    x = s["qkv"].float().view(s["tokens"], hq + 2 * hkv, hd)
    qk, v = x[:, : hq + hkv], x[:, hq + hkv:]
    gain = torch.cat([s["q_gain"].expand(hq, hd), s["k_gain"].expand(hkv, hd)])
    y = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * gain
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = y[..., : hd // 2], y[..., hd // 2:]
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    at, off = s["table"].long()[s["seq"], s["slot"] // page], s["slot"] % page
    s["k"][at, :, off] = y[:, hq:].to(s["k"].dtype)
    s["v"][at, :, off] = v.to(s["v"].dtype)
    if s["mass"] is not None:
        s["mass"][at, :, off] = 0.0
    return y[:, :hq].to(s["qkv"].dtype), s["k"], s["v"], s["mass"]


def _plain_evict(s):
    c = s["case"]
    n, hkv, page, keep = c["seqs"], c["hkv"], c["page"], c["keep"]
    length = int(s["table"].shape[1]) * page
    m = _gathered(s["mass"], s["table"], length)
    lens = s["lens"].long()[:, None, None]
    j = torch.arange(length, device=DEV)
    sure = (j < c["sinks"]) | (j >= lens - c["recent"])
    m = m.masked_fill(sure, math.inf).masked_fill(j >= lens, -math.inf)
    order = m.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    live = torch.arange(order.shape[-1], device=DEV) < lens
    kept = torch.where(live, order, length).sort(dim=-1).values
    kept = torch.nn.functional.pad(kept, (0, keep - kept.shape[-1]), value=length)
    live = kept < length
    src, h, d = kept.clamp_max(length - 1), torch.arange(hkv, device=DEV)[:, None], torch.arange(keep, device=DEV)
    b = torch.arange(n, device=DEV)[:, None, None]
    from_page, to_page = s["table"].long()[b, src // page], s["dst"].long()[:, d // page][:, None].expand_as(kept)
    hh, to_off = h.expand_as(kept), (d % page).expand_as(kept)
    to = (to_page[live], hh[live], to_off[live])
    at = (from_page[live], hh[live], (src % page)[live])
    s["k"][to], s["v"][to], s["mass"][to] = s["k"][at], s["v"][at], s["mass"][at]
    return s["lens"].clamp_max(keep), torch.where(live, kept, -1).int(), s["k"], s["v"], s["mass"]


# ------------------------------------------------------------------ one pass

def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        ops = _ops()
        heads = (c["hq"], c["hkv"], c["hd"], c["page"])
        if kind == "append":
            q = ops.paged_append(*heads, EPS)(s["qkv"], s["q_gain"], s["k_gain"], s["inv_freq"], s["positions"],
                                              s["starts"], s["lens"], s["table"], s["k"], s["v"], mass=s["mass"])
            return q, s["k"], s["v"], s["mass"]
        if kind == "attend":
            lse = torch.empty(s["tokens"], c["hq"], device=DEV)
            out = ops.paged_attention(*heads, s["scale"], c["window"], c["sinks"])(
                s["q"], s["k"], s["v"], s["table"], s["starts"], s["lens"], lse=lse)
            return out, lse
        if kind == "mass":
            return ops.paged_attention_mass(*heads, s["scale"], c["window"], c["sinks"])(
                s["q"], s["lse"], s["k"], s["table"], s["starts"], s["lens"], s["mass"])
        lens, kept = ops.paged_evict(c["hkv"], c["hd"], c["page"], c["keep"], c["sinks"], c["recent"])(
            s["k"], s["v"], s["mass"], s["table"], s["lens"], s["dst"])
        return lens, kept, s["k"], s["v"], s["mass"]
    if kind == "append":
        return _plain_append(s)
    if kind == "attend":
        return _plain_attend(s)
    if kind == "mass":
        return _plain_mass(s)
    return _plain_evict(s)


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, hd, page = case["hq"], case["hkv"], case["hd"], case["page"]
    gr, kind = hq // hkv, case["kind"]
    table, starts, lens = (s[k].tolist() for k in ("table", "starts", "lens"))

    def rows(pool, u, h, length):
        """Slots 0..length of one head of sequence u, in 64 bits."""
        return pool[torch.tensor(table[u], device=DEV), h].flatten(0, 1)[:length].double()

    if kind == "append":
        x = s["qkv"].double().view(-1, hq + 2 * hkv, hd)
        turn = torch.polar(torch.ones((), device=DEV, dtype=torch.float64),
                           s["positions"].double()[:, None] * s["inv_freq"].double())
        q = torch.empty(x.shape[0], hq, hd, device=DEV, dtype=torch.float64)
        k, v = s["k"].double(), s["v"].double()
        mass = None if s["mass"] is None else s["mass"].double()
        for h in range(hq + hkv):
            y = x[:, h] / (x[:, h].pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt()
            y = y * (s["q_gain"] if h < hq else s["k_gain"]).double()
            z = torch.complex(y[:, : hd // 2], y[:, hd // 2:]) * turn
            x[:, h] = torch.cat([z.real, z.imag], -1)
        q[:] = x[:, :hq]
        for u in range(case["seqs"]):
            n = starts[u + 1] - starts[u]
            j = np.arange(lens[u] - n, lens[u])
            pg, off = torch.from_numpy(np.asarray(table[u])[j // page]).to(DEV), torch.from_numpy(j % page).to(DEV)
            mine = x[starts[u]: starts[u + 1]]
            k[pg, :, off], v[pg, :, off] = mine[:, hq: hq + hkv], mine[:, hq + hkv:]
            if mass is not None:
                mass[pg, :, off] = 0.0
        return q, k, v, mass
    if kind == "evict":
        mass = s["mass"].cpu().numpy()
        k, v, m64 = s["k"].double(), s["v"].double(), s["mass"].double()
        kept = np.full((case["seqs"], hkv, case["keep"]), -1, np.int32)
        for u in range(case["seqs"]):
            for h in range(hkv):
                w = mass[table[u], h].reshape(-1)[: lens[u]]
                n = min(lens[u], case["keep"])
                sure = np.zeros(lens[u], bool)
                sure[: case["sinks"]] = True
                sure[max(0, lens[u] - case["recent"]):] = True
                best = np.lexsort((np.arange(lens[u]), -w, ~sure))[:n]
                kept[u, h, :n] = np.sort(best)
                j, d = kept[u, h, :n], np.arange(n)
                pt, dt = np.asarray(table[u]), s["dst"][u].cpu().numpy()
                a, b = torch.from_numpy(pt[j // page]).to(DEV), torch.from_numpy(j % page).to(DEV)
                y, z = torch.from_numpy(dt[d // page]).to(DEV), torch.from_numpy(d % page).to(DEV)
                k[y, h, z], v[y, h, z], m64[y, h, z] = k[a, h, b], v[a, h, b], m64[a, h, b]
        return np.minimum(np.asarray(lens, np.int32), case["keep"]).astype(np.int32), kept, k, v, m64
    t = starts[-1]
    out = torch.zeros(t, hq, hd, device=DEV, dtype=torch.float64)
    lse = torch.full((t, hq), -math.inf, device=DEV, dtype=torch.float64)
    mass = s["mass"].double() if kind == "mass" else None
    for u in range(case["seqs"]):
        n = starts[u + 1] - starts[u]
        p = torch.arange(lens[u] - n, lens[u], device=DEV)[:, None]
        j = torch.arange(lens[u], device=DEV)
        hide = j > p
        if case["window"]:
            hide = hide | ((j <= p - case["window"]) & (j >= case["sinks"]))
        for h in range(hkv):
            k = rows(s["k"], u, h, lens[u]).t().contiguous()
            got = torch.zeros(lens[u], device=DEV, dtype=torch.float64)
            for a in range(h * gr, h * gr + gr):
                x = torch.mm(s["q"][starts[u]: starts[u + 1], a].double(), k) / math.sqrt(hd)
                x[hide] = -math.inf
                if kind == "mass":
                    got += torch.exp(x - s["lse"][starts[u]: starts[u + 1], a].double()[:, None]).sum(0)
                else:
                    lse[starts[u]: starts[u + 1], a] = torch.logsumexp(x, 1)
                    out[starts[u]: starts[u + 1], a] = torch.mm(torch.softmax(x, 1), rows(s["v"], u, h, lens[u]))
            if kind == "mass":
                pad = torch.nn.functional.pad(got, (0, len(table[u]) * page - lens[u])).view(-1, page)
                mass[torch.tensor(table[u], device=DEV), h] += pad
    return mass if kind == "mass" else (out, lse)
