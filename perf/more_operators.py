"""Cases of the 8-bit projections and of the sampler that draws from their logits.

Each case is one call of ``soraku_amd.ops``:

* ``rows``    the rows of a matrix as 8-bit codes with a scale each
              (``ops.int8_rows``): how a program makes its weights' codes;
* ``linear``  a projection whose weights are such codes: the activations' rows,
              normalised or not, become codes on the way, the product is summed in
              whole numbers, then scales, bias, SwiGLU, residual (``ops.int8_linear``);
* ``sample``  one token for each row of logits from given uniform draws:
              classifier-free guidance, allowed ids, temperature, top-k, top-p and
              min-p, all by row (``ops.sample_rows``).

``own`` chooses between those calls and the plain form: elementary torch
operations in 32 bits, in 64 where a value next to a border decides (a code
between two whole numbers, a draw between two tokens).

The definitions fix what is rounded, so that codes and tokens are determined: a
normalised row enters its codes as fp32(x * gain), without the norm's factor,
which all of the row shares and which goes into the scale; codes are the nearest
whole numbers (ties to even) of 127 t / max|t|, exactly; logits are merged and divided
by the temperature in 32 bits, each operation rounded, and weights are summed in 64.

Sizes are the package's trunk shapes (projections of 1,024 and 2,048 by 2,048 to 12,288 and
of 6,144 by 2,048), its codebooks of 2,051, its text vocabulary of 151,936, and,
drawn, others down to 16 by 16.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6           # the trunk's norm
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

def _rows(rows, k, bf16=False):
    return dict(kind="rows", rows=rows, k=k, bf16=bf16)


def _linear(rows, n, k, *, bf16=False, norm=False, swiglu=False, bias=False, residual=False):
    return dict(kind="linear", rows=rows, n=n, k=k, bf16=bf16, norm=norm, swiglu=swiglu, bias=bias, residual=residual)


def _sample(rows, v, *, bf16=False, cfg=False, temp=0.9, top_k=0, top_p=0.0, min_p=0.0, allowed=False, spread=2.5):
    return dict(kind="sample", rows=rows, v=v, bf16=bf16, cfg=cfg, temp=temp, top_k=top_k, top_p=top_p, min_p=min_p,
                allowed=allowed, spread=spread)


def listed():
    return [
        # a layer's gate and up matrices at load time
        dict(_rows(12288, 2048, bf16=True), name="rows_gate_up_bf16"),
        # all sixteen codebooks, FP32 as checkpoints hold them
        dict(_rows(32816, 1024), name="rows_codebooks_f32"),
        # one codebook's classifier for one row: all latency, an odd number of outputs
        dict(_linear(1, 2051, 1024, bias=True), name="linear_classifier_1row"),
        # q, k and v of a CFG pair's single tokens, the layer's norm in front
        dict(_linear(2, 4096, 2048, norm=True), name="linear_pair_qkv"),
        # gate and up, then down, of a frame of 16 utterances with CFG
        dict(_linear(32, 6144, 2048, bf16=True, norm=True, swiglu=True), name="linear_step_gate_up"),
        dict(_linear(32, 2048, 6144, residual=True), name="linear_step_down_f32"),
        # q, k and v of a CFG pair's prefix, FP32 activations
        dict(_linear(774, 4096, 1024, norm=True), name="linear_prompt_qkv_f32"),
        # a serving batch's prefixes: gate and up, and down of a ragged number of tokens
        dict(_linear(7680, 6144, 2048, bf16=True, norm=True, swiglu=True), name="linear_prompts_gate_up"),
        dict(_linear(5999, 2048, 6144, bf16=True, residual=True), name="linear_prompts_down"),
        # a codebook step of 16 utterances with CFG, the reference's filters
        dict(_sample(16, 2051, cfg=True, top_k=50, top_p=0.95, allowed=True), name="sample_codes_16utts"),
        # one row over the text vocabulary
        dict(_sample(1, 151936, temp=0.8, top_p=0.95, min_p=0.02), name="sample_text_1row"),
        # a serving batch over the text vocabulary, flat: tens of thousands of ids are kept
        dict(_sample(64, 151936, bf16=True, temp=1.0, top_p=0.9), name="sample_text_64rows_bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["rows", "linear", "linear", "linear", "sample", "sample"])
    top = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        bf16 = rng.random() < 0.5
        if kind == "rows":
            c = _rows(_log_int(rng, 1, 32816), _log_int(rng, 16, 8192), bf16)
        elif kind == "linear":
            n, k = rng.choice([(4096, 1024), (4096, 2048), (2048, 6144), (1024, 2048), (2051, 1024), (6144, 2048)] +
                              [(_log_int(rng, 16, 12288), _log_int(rng, 16, 8192)) for _ in range(4)])
            c = _linear(_log_int(rng, 1, 7680), n, k, bf16=bf16, norm=rng.random() < 0.5, swiglu=rng.random() < 0.3,
                        bias=rng.random() < 0.3, residual=rng.random() < 0.4)
        else:
            c = _sample(_log_int(rng, 1, 256), rng.choice([2051, 151936, _log_int(rng, 40, 151936)]), bf16=bf16,
                        cfg=rng.random() < 0.4, temp=rng.choice([0.0, 0.7, 1.0, rng.uniform(0.3, 1.5)]),
                        top_k=rng.choice([0, 0, 1, 50, _log_int(rng, 2, 2000)]),
                        top_p=rng.choice([0.0, 0.95, rng.uniform(0.05, 0.99)]),
                        min_p=rng.choice([0.0, 0.0, 0.05, rng.uniform(0.001, 0.5)]), allowed=rng.random() < 0.3,
                        spread=rng.choice([1.0, 2.5, 6.0]))
        if _cost(c) <= top:
            return c


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 1.2e15


def work(case):
    b = 2 if case["bf16"] else 4
    if case["kind"] == "rows":
        r, k = case["rows"], case["k"]
        return {"bytes": r * (k * (b + 1) + 4), "flops": 2 * r * k}
    if case["kind"] == "sample":
        r, v = case["rows"], case["v"]
        words = r * -(-v // 32)
        return {"bytes": r * (v * b * (2 if case["cfg"] else 1) + 44) + (4 * words if case["allowed"] else 0), "flops": 4 * r * v}
    m, n, k = case["rows"], case["n"], case["k"]
    both = n * (2 if case["swiglu"] else 1)
    return {"bytes": m * k * b + (4 * k if case["norm"] else 0) + both * (k + (8 if case["bias"] else 4)) +
            m * n * b * (2 if case["residual"] else 1), "flops": 2 * m * both * k}


# ------------------------------------------------------------------ inputs

def _padded(k):
    """Codes of a row of k: up to whole groups of 128, zeros behind."""
    return -(-k // 128) * 128


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 53)
    kind, dt = case["kind"], torch.bfloat16 if case["bf16"] else torch.float32

    def rand(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV).mul_(scale).to(dtype)

    s = dict(case=case)
    if kind == "rows":
        # weights as an initialiser leaves them, rows of unequal size
        s["x"] = (rand(case["rows"], case["k"], scale=0.02) * rand(case["rows"], 1, scale=0.3).exp_()).to(dt)
        return s
    if kind == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        both = n * (2 if case["swiglu"] else 1)
        # activations of unequal rows, a few channels much larger than the others
        x = rand(m, k).mul_(rand(m, 1, scale=0.3).exp_())
        x[:, torch.randperm(k, generator=g, device=DEV)[: max(1, k // 256)]] *= 8.0
        s["x"] = x.to(dt)
        s["codes"], s["scales"] = _plain_rows(rand(both, k, scale=k ** -0.5))
        s["gain"] = rand(k, scale=0.1).add_(1.0) if case["norm"] else None
        s["bias"] = rand(both, scale=0.5) if case["bias"] else None
        s["residual"] = rand(m, n, dtype=dt) if case["residual"] else None
        return s
    r, v = case["rows"], case["v"]
    base = rand(r, 1, v, scale=case["spread"])
    s["logits"] = (base + rand(r, 2, v, scale=0.3 * case["spread"])).to(dt) if case["cfg"] else base[:, 0].to(dt)

    def uniform(*shape, dtype=torch.float32):
        return torch.rand(*shape, generator=g, device=DEV, dtype=dtype)

    s["u"] = uniform(r, dtype=torch.float64)
    # every row has its own parameters; one in eight is greedy
    s["temperature"] = uniform(r).mul_(0.2).add_(0.9).mul_(case["temp"]).mul_((uniform(r) > 0.125 if r > 1 else 1))
    s["top_k"] = (uniform(r).mul_(0.5).add_(0.75) * case["top_k"]).ceil().int() if case["top_k"] else None
    s["top_p"] = 1.0 - (1.0 - case["top_p"]) * (0.75 + 0.5 * uniform(r)) if case["top_p"] else None
    if case["top_p"]:
        s["top_p"] = s["top_p"].clamp_min_(0.01)
    s["min_p"] = uniform(r).mul_(0.5).add_(0.75).mul_(case["min_p"]) if case["min_p"] else None
    s["cfg_scale"] = uniform(r).add_(1.0) if case["cfg"] else None
    s["allowed"] = None
    if case["allowed"]:
        # a few ids blocked, as BOS, PAD and EOS are
        ok = uniform(r, -(-v // 32), 32) > 0.01
        bits = (ok.long() << torch.arange(32, device=DEV)).sum(-1)
        s["allowed"] = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).int()
    return s


# ------------------------------------------------------------------ plain form

def _plain_rows(t):
    """Codes [rows, whole groups of 128] and scales of rows in 32 bits."""
    top = t.abs().amax(-1, keepdim=True)
    q = (t.double() * 127.0 / top.double()).nan_to_num_(0.0).round_().to(torch.int8)
    return torch.nn.functional.pad(q, (0, _padded(t.shape[1]) - t.shape[1])), (top / 127.0).squeeze(-1)


def _plain_linear(s):
    c = s["case"]
    t = x = s["x"].float()
    if c["norm"]:
        t = x * s["gain"]
    q, scale = _plain_rows(t)
    if c["norm"]:
        scale = scale * torch.rsqrt(x.square().mean(-1) + EPS)
    y = torch.matmul(q.float(), s["codes"].float().t())
    y = y * scale[:, None] * s["scales"]
    if c["bias"]:
        y = y + s["bias"]
    if c["swiglu"]:
        y = y[:, : c["n"]] * torch.sigmoid(y[:, : c["n"]]) * y[:, c["n"]:]
    if c["residual"]:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_sample(s):
    c, v = s["case"], s["case"]["v"]
    x = s["logits"].float()
    if c["cfg"]:
        x = x[:, 1] + s["cfg_scale"][:, None] * (x[:, 0] - x[:, 1])
    ok = x.isfinite()
    if c["allowed"]:
        bit = s["allowed"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32) & 1
        ok &= bit.flatten(1)[:, :v] != 0
    hot = s["temperature"][:, None] > 0
    x = torch.where(hot, (x / s["temperature"][:, None]).clamp(-3.4028234e38, 3.4028234e38), x)
    x, order = x.masked_fill_(~ok, -math.inf).sort(dim=-1, descending=True, stable=True)
    n = ok.sum(-1, keepdim=True)
    at = torch.arange(v, device=DEV)
    if c["top_k"]:
        k = s["top_k"].long()[:, None]
        cut = x.gather(1, (k - 1).clamp(0, v - 1))
        n = torch.where((k > 0) & (k < n), (x >= cut).sum(-1, keepdim=True), n)
    w = (x.double() - x[:, :1].double()).exp_().masked_fill_(at >= n, 0.0)
    sums = w.cumsum(-1)
    keep = n
    if c["top_p"]:
        p = s["top_p"].double()[:, None]
        over = (sums <= p * sums[:, -1:]).sum(-1, keepdim=True) + 1
        keep = torch.where((p > 0) & (p < 1), torch.minimum(over, n), n)
    if c["min_p"]:
        keep = torch.minimum(keep, (w >= s["min_p"].double()[:, None]).sum(-1, keepdim=True))
    keep = torch.where(hot, keep, torch.ones_like(keep))
    total = sums.gather(1, keep - 1)
    j = torch.minimum((sums <= s["u"][:, None] * total).sum(-1, keepdim=True), keep - 1)
    logprob = w.gather(1, j).log_() - total.log()
    return order.gather(1, j)[:, 0], logprob[:, 0].float(), keep[:, 0].int()


# ------------------------------------------------------------------ one pass

def run(s):
    c = s["case"]
    if c["kind"] == "rows":
        codes, scales = _ops().int8_rows(c["k"])(s["x"]) if own else _plain_rows(s["x"].float())
        # what the codes stand for
        return torch.mul(codes[:, : c["k"]], scales[:, None]), scales
    if c["kind"] == "linear":
        if not own:
            return _plain_linear(s)
        project = _ops().int8_linear(c["n"], c["k"], act="swiglu" if c["swiglu"] else None, eps=EPS if c["norm"] else None)
        return project(s["x"], s["codes"], s["scales"], gain=s["gain"], bias=s["bias"], residual=s["residual"])
    if not own:
        return _plain_sample(s)
    logprob = torch.empty(c["rows"], device=DEV)
    kept = torch.empty(c["rows"], device=DEV, dtype=torch.int32)
    token = _ops().sample_rows(c["v"], cfg=c["cfg"])(
        s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
        cfg_scale=s["cfg_scale"], allowed=s["allowed"], logprob=logprob, kept=kept)
    return token, logprob, kept


# ------------------------------------------------------------------ 64 bits

def _exact_codes(t):
    """What rows stand for and their scales; t in 64 bits, its values those of 32."""
    top = t.abs().max(1, keepdim=True).values
    lo = torch.floor(127.0 * t / top)
    frac = 254.0 * t - (2.0 * lo + 1.0) * top            # exact: above, at or below the middle
    q = torch.where((frac > 0) | ((frac == 0) & (lo % 2 != 0)), lo + 1, lo)
    q = torch.where(top > 0, q, torch.zeros_like(q))
    return q, top[:, 0] / 127.0


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rows":
        q, scale = _exact_codes(s["x"].double())
        return q * scale[:, None], scale
    if case["kind"] == "linear":
        x = s["x"].double()
        # fp32(x * gain) is part of the definition
        q, scale = _exact_codes((x * s["gain"].double()).float().double() if case["norm"] else x)
        if case["norm"]:
            scale = scale / (x.pow(2).sum(1) / case["k"] + EPS).sqrt()
        n, k = case["n"], case["k"]

        def side(rows):
            w = s["codes"][rows, :k].double() * s["scales"][rows].double()[:, None]
            y = torch.mm(q * scale[:, None], w.t().contiguous())
            return y if s["bias"] is None else y + s["bias"][rows].double()

        y = side(slice(0, n))
        if case["swiglu"]:
            y = y / (1.0 + torch.exp(-y)) * side(slice(n, 2 * n))
        return y if s["residual"] is None else y + s["residual"].double()
    tokens, logprobs, kept = [], [], []
    for r in range(case["rows"]):
        # 32-bit merging and division are part of the definition
        z = s["logits"][r].float()
        if case["cfg"]:
            z = z[1] + s["cfg_scale"][r] * (z[0] - z[1])
        t = float(s["temperature"][r])
        z = z / s["temperature"][r] if t > 0 else z
        ids = torch.arange(case["v"], device=DEV)
        if case["allowed"]:
            word = s["allowed"][r].long()[ids // 32]
            ids = ids[(word >> (ids % 32)) % 2 == 1]
        val = z[ids].double()
        # a stable sort in 64 bits, largest first
        order = torch.argsort(-val, stable=True)
        ids, val = ids[order], val[order]
        if t <= 0:
            n = 1
        else:
            n = val.numel()
            k = int(s["top_k"][r]) if case["top_k"] else 0
            if 0 < k < n:
                n = int(torch.searchsorted(-val, -val[k - 1], right=True))
            mass = torch.exp(val - val[0])[:n]
            run_sum = mass.cumsum(0)
            low = math.log(float(s["min_p"][r])) if case["min_p"] else -math.inf
            if case["top_p"]:
                n = min(n, int(torch.searchsorted(run_sum, float(s["top_p"][r]) * float(run_sum[-1]), right=True)) + 1)
            n = min(n, int(torch.searchsorted(val[0] - val, torch.tensor(-low, device=DEV, dtype=torch.float64), right=True)))
        run_sum = torch.exp(val[:n] - val[0]).cumsum(0)
        j = min(n - 1, int(torch.searchsorted(run_sum, float(s["u"][r]) * float(run_sum[-1]), right=True)))
        tokens.append(int(ids[j]))
        logprobs.append(float(val[j] - val[0]) - math.log(float(run_sum[-1])) if t > 0 else 0.0)
        kept.append(n)
    return (torch.tensor(tokens), torch.tensor(logprobs, dtype=torch.float64), torch.tensor(kept, dtype=torch.int32))
