"""A decode step of trunk layers and classifier in 8 bits, operator by operator: projections with codes, the cache in
pages between them, ids drawn by row from the logits.  Each operator is held to its formula on what the one before it
left; the whole step, captured, gives what the calls one by one give."""

import numpy as np
import pytest
import torch

import draw_ref
import int8_ref as ref

pytestmark = pytest.mark.gpu

D, HQ, HKV, HD, INNER, V, LAYERS, UTTS, PAGE = 192, 6, 2, 32, 320, 515, 2, 3, 16
EPS = 1e-6
ROWS = 2 * UTTS                                      # cond and uncond of each


class Step:
    """Weights, caches and the calls of one step."""

    def __init__(self, ops, dev, dtype):
        g = torch.Generator().manual_seed(5)
        rand = lambda *s, scale=1.0: torch.randn(*s, generator=g) * scale  # noqa: E731
        self.ops, self.dev, self.dtype, self.trace = ops, dev, dtype, None
        self.w = {}

        def weight(name, n, k):
            self.w[name] = ops.int8_rows(k)(rand(n, k, scale=k ** -0.5).to(dev))
        for i in range(LAYERS):
            weight(f"qkv{i}", (HQ + 2 * HKV) * HD, D)
            weight(f"o{i}", D, HQ * HD)
            weight(f"gate_up{i}", 2 * INNER, D)
            weight(f"down{i}", D, INNER)
        weight("head", V, D)
        self.gain = {n: (1 + rand(D, scale=0.1)).to(dev) for n in [f"{p}{i}" for i in range(LAYERS) for p in "am"] + ["f"]}
        self.qk = [(1 + rand(HD, scale=0.1)).to(dev) for _ in range(2)]
        self.bias = rand(V, scale=0.2).to(dev)
        self.embed = rand(V, D).to(dev).to(dtype)
        self.freq = (1e4 ** (-torch.arange(0, HD, 2) / HD)).float().to(dev)
        width = 3
        order = torch.randperm(ROWS * width * LAYERS, generator=g).int()
        self.tables = [order[i * ROWS * width: (i + 1) * ROWS * width].view(ROWS, width).to(dev) for i in range(LAYERS)]
        kv = torch.bfloat16 if dtype == torch.bfloat16 else torch.float32
        self.k = torch.zeros(ROWS * width * LAYERS, HKV, PAGE, HD, device=dev, dtype=kv)
        self.v = torch.zeros_like(self.k)
        self.starts = torch.arange(ROWS + 1, device=dev, dtype=torch.int32)
        self.lens = torch.zeros(ROWS, device=dev, dtype=torch.int32)
        self.ids = torch.tensor([3, 100, 514], device=dev)
        self.u = torch.zeros(UTTS, device=dev, dtype=torch.float64)
        full = lambda c, t=torch.float32: torch.full((UTTS,), c, device=dev, dtype=t)  # noqa: E731
        self.how = dict(temperature=torch.tensor([0.9, 0.0, 1.2], device=dev), top_k=torch.tensor([50, 0, 7], device=dev, dtype=torch.int32),
                        top_p=full(0.95), min_p=full(0.01), cfg_scale=full(1.5))
        self.logprob, self.kept = full(0.0), full(0, torch.int32)

    def linear(self, name, x, n, act=None, gain=None, bias=None, residual=None):
        codes, scales = self.w[name]
        eps = None if gain is None else EPS
        y = self.ops.int8_linear(n, x.shape[1], act=act, eps=eps)(x, codes, scales, gain=gain, bias=bias, residual=residual)
        if self.trace is not None:
            np_ = lambda t: None if t is None else t.float().cpu().numpy()  # noqa: E731
            want, off = ref.linear(np_(x), codes.cpu().numpy(), np_(scales), np_(gain), eps, np_(bias), np_(residual), act == "swiglu",
                                   x.dtype == torch.bfloat16)
            half = ref.HALF_STEP[str(x.dtype)[6:]]
            err = np.abs(y.double().cpu().numpy() - want)
            assert (err <= off + (np.abs(want) + off) * half + 2.0 ** -133).all(), name
            self.trace.append(name)
        return y

    def __call__(self):
        ops = self.ops
        self.lens += 1
        at = self.lens - 1
        h = self.embed[self.ids].repeat_interleave(2, 0).contiguous()
        for i in range(LAYERS):
            qkv = self.linear(f"qkv{i}", h, (HQ + 2 * HKV) * HD, gain=self.gain[f"a{i}"])
            q = ops.paged_append(HQ, HKV, HD, PAGE, EPS)(qkv, *self.qk, self.freq, at, self.starts, self.lens, self.tables[i], self.k, self.v)
            o = ops.paged_attention(HQ, HKV, HD, PAGE)(q, self.k, self.v, self.tables[i], self.starts, self.lens)
            h = self.linear(f"o{i}", o.view(ROWS, HQ * HD), D, residual=h)
            a = self.linear(f"gate_up{i}", h, INNER, act="swiglu", gain=self.gain[f"m{i}"])
            h = self.linear(f"down{i}", a, D, residual=h)
        logits = self.linear("head", h, V, gain=self.gain["f"], bias=self.bias).view(UTTS, 2, V)
        ops.sample_rows(V, cfg=True)(logits, self.u, out=self.ids, logprob=self.logprob, kept=self.kept, **self.how)
        if self.trace is not None:
            x = draw_ref.merge(logits.float().cpu().numpy(), self.how["cfg_scale"].cpu().numpy())
            for r in range(UTTS):
                p = {k: v[r].item() for k, v in self.how.items() if k != "cfg_scale"}
                tok, lp, n, margin, sure = draw_ref.row(x[r], float(self.u[r]), **p)
                assert sure and margin > draw_ref.safe(V) and int(self.ids[r]) == tok and int(self.kept[r]) == n
                assert abs(float(self.logprob[r]) - lp) <= abs(lp) * 2.0 ** -24 + 1e-8
        return logits


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_by_operators(hip_device, dtype):
    from soraku_amd import ops

    draws = torch.rand(12, UTTS, dtype=torch.float64, generator=torch.Generator().manual_seed(8)).to(hip_device)
    eager = Step(ops, hip_device, dtype)
    eager.trace = []
    want = []
    for t in range(12):
        eager.u.copy_(draws[t])
        logits = eager()
        want.append((eager.ids.clone(), logits.clone(), eager.logprob.clone()))
    assert len(eager.trace) == 12 * (4 * LAYERS + 1) and len({tuple(w[0].tolist()) for w in want}) > 3

    s = Step(ops, hip_device, dtype)
    s()                                              # first calls load code; then from the beginning again
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        logits = s()
    s.ids.copy_(torch.tensor([3, 100, 514]))
    s.lens.zero_()
    for t in range(12):
        s.u.copy_(draws[t])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(s.ids, want[t][0]) and torch.equal(logits, want[t][1]) and torch.equal(s.logprob, want[t][2])
