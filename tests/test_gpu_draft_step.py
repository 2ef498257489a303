"""The operators of a serving step whose sequences share a prefix and verify
drafted tokens, run one after the other on what the one before left: normalised
and rotated q and k, the rows stored at the step's slots, attention over them,
the drafts verified on its outputs (taken as logits). Each stage is checked as
in its own tests, from what it was given."""
import numpy as np
import pytest
import torch

from test_gpu_prefix import BATCH, LLAMA, QWEN, Step
from test_gpu_qk_norm import Case
from test_gpu_verify import plain

pytestmark = pytest.mark.gpu

SEQS = [(0, 20, 30 + 7 * i, 1 + i % 5) for i in range(11)] + [(1, 70, 9, 2), (1, 66, 40, 1), (2, 0, 5, 5), (2, 0, 1, 1)]


class Flow:
    def __init__(self, seqs, heads, kv="bf16", seed=0):
        from llm_engine_amd import kernels
        self.step = s = Step(seqs, heads, "bf16", kv, seed=seed)
        plan = kernels.Plan(s.slices, *heads, s.bs, s.k.dtype).upload()
        n = sum(s.rows)
        self.norm = c = Case(n, heads, "bf16", kv, max_pos=2048, seed=seed)
        c.pos, c.slots, c.k, c.v = plan.dev_array("positions"), plan.dev_array("slots"), s.k, s.v
        self.cu = np.concatenate([[0], np.cumsum([r - 1 for r in s.rows])]).astype(np.int32)
        self.vocab, self.max_drafts = s.H * s.d, max(s.rows) - 1
        g = torch.Generator(device=s.dev)
        g.manual_seed(seed + 1)
        drafts, self.cu_dev = int(self.cu[-1]), torch.from_numpy(self.cu).to(s.dev)
        self.probs = torch.softmax(torch.randn(drafts, self.vocab, device=s.dev, generator=g), -1)
        self.tokens = torch.multinomial(self.probs, 1, generator=g)[:, 0].to(torch.int32)
        self.au = torch.rand(drafts, device=s.dev, generator=g)
        self.su = torch.rand(len(seqs), device=s.dev, generator=g)

    def verify(self, logits, **kw):
        from llm_engine_amd import kernels
        return kernels.verify_drafts(logits, self.cu_dev, self.tokens, self.au, self.su, self.max_drafts,
                                     draft_probs=self.probs, **kw)

    def run(self, **kw):
        self.step.q = self.norm.run(**kw)
        o = self.step.run(**kw)
        return (self.step.q, o) + self.verify(o, **kw)


@pytest.mark.parametrize("heads", [QWEN, LLAMA, (16, 2, 128)])
@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_stages(gpu, heads, kv):
    f = Flow(SEQS, heads, kv, seed=3)
    f.step.q = f.norm.check()
    o = f.step.run()
    f.step.check(o)
    out, acc = f.verify(o)
    want, n = plain(o.double().cpu().numpy(), f.cu.tolist(), f.tokens.tolist(), f.au.double().cpu().numpy(),
                    f.su.double().cpu().numpy(), f.max_drafts, f.probs.double().cpu().numpy(), None)
    assert acc.tolist() == n.tolist() and (out.cpu().numpy() == want).all()


def test_one_graph(gpu):
    """The step captured once and replayed with other projections: every replay
    gives what the eager calls give, and leaves the same cache."""
    f = Flow(SEQS, QWEN, seed=4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    f.run(stream=stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        held = f.run()
    rows = f.norm.slots.long()
    for i in range(3):
        f.norm.qkv.copy_(torch.randn(f.norm.qkv.shape, device=f.step.dev,
                                     generator=torch.Generator(device=f.step.dev).manual_seed(i)))
        eager = [t.clone() for t in f.run()]
        cache = f.step.k.clone(), f.step.v.clone()
        f.step.k[rows], f.step.v[rows] = 0, 0
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))
        assert torch.equal(f.step.k, cache[0]) and torch.equal(f.step.v, cache[1])


def busy(dev):
    """20 ms of work on the current stream."""
    a = torch.ones(4096, 4096, device=dev)
    for _ in range(20):
        a @ a


def test_temporaries_on_another_stream(gpu):
    """Outputs and workspaces that the calls make come from the pool of the stream
    they launch on: what the current stream has yet to do to freed tensors of
    their sizes does not reach them."""
    f = Flow(BATCH, QWEN, seed=5)
    want = f.run()
    from llm_engine_amd import kernels
    sizes = [t.numel() * t.element_size() for t in want]
    sizes += [f.step.plan.workspace_size(),
              kernels.verify_drafts_workspace_size(len(f.cu) - 1, int(f.cu[-1]), f.vocab)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy(f.step.dev)
    for _ in range(2):
        old = [torch.empty(n, dtype=torch.uint8, device=f.step.dev) for n in sizes for _ in range(3)]
        for t in old:
            t.fill_(255)
        del old, t
    got = f.run(stream=stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_plans_dropped_while_their_copies_wait(gpu):
    """A loop that packs, uploads and drops a plan per step, ahead of the device."""
    from llm_engine_amd import kernels
    s = Step([(0, 20, 40 + i, 1) for i in range(8)], QWEN, seed=6)
    orders = [np.roll(np.arange(8), i) for i in range(6)]  # slice i's rows are q's row i
    slices = [[s.slices[j] for j in o] for o in orders]

    def outs():
        r = []
        for o in slices:
            plan = kernels.PrefixPlan(o, *QWEN, 16, torch.bfloat16).upload()
            r.append(kernels.shared_prefix_attention(s.q, s.k, s.v, plan, s.scale))
            del plan
        return r

    want = []
    for o in slices:
        plan = kernels.PrefixPlan(o, *QWEN, 16, torch.bfloat16).upload()
        want.append(kernels.shared_prefix_attention(s.q, s.k, s.v, plan, s.scale))
        torch.cuda.synchronize()
    busy(s.dev)
    got = outs()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_upload_through_the_abi(gpu):
    """le_prefix_plan_upload: the same device copy."""
    import ctypes

    from llm_engine_amd import _lib, kernels
    s = Step(BATCH, QWEN, seed=7)
    want = s.run()
    plan = kernels.PrefixPlan(s.slices, *QWEN, 16, torch.bfloat16)
    buf = torch.empty(int(plan.plan.bytes), dtype=torch.uint8, device=s.dev)
    raw = torch.cuda.current_stream().cuda_stream
    assert _lib.load().le_prefix_plan_upload(ctypes.byref(plan.plan), plan.host.data_ptr(), buf.data_ptr(), raw) == 0
    plan.device_buf = buf
    assert torch.equal(kernels.shared_prefix_attention(s.q, s.k, s.v, plan, s.scale), want)


def test_empty_steps(gpu):
    """No rows, no sequences: nothing is launched, nothing changes."""
    from llm_engine_amd import kernels
    f = Flow(BATCH, QWEN, seed=8)
    c, k = f.norm, f.step.k.clone()
    q = kernels.qk_norm_rope_store_kv(c.qkv[:0], c.pos, c.slots, c.cos, c.sin, c.qw, c.kw, c.eps, *QWEN, c.k, c.v)
    plan = kernels.PrefixPlan([], *QWEN, 16, torch.bfloat16).upload()
    out = kernels.shared_prefix_attention(q, f.step.k, f.step.v, plan, 1.0)
    none = torch.zeros(0, device=f.step.dev)
    tokens, n = kernels.verify_drafts(torch.zeros(0, 50, device=f.step.dev), f.cu_dev[:1], f.tokens[:0], none, none, 3)
    assert q.shape == out.shape == (0, 14 * 64) and tokens.shape == (0, 4) and n.shape == (0,)
    torch.cuda.synchronize()
    assert torch.equal(f.step.k, k)


def test_two_steps_at_once(gpu):
    """Two steps, each on a stream of its own, not waiting for each other: each
    gives what it gives alone."""
    flows = [Flow(SEQS, QWEN, seed=9), Flow([(0, 30, 20 + i % 30, 1 + i % 2) for i in range(90)], LLAMA, seed=10)]
    want = [[t.clone() for t in f.run()] for f in flows]
    streams = [torch.cuda.Stream() for _ in flows]
    torch.cuda.synchronize()
    got = [[] for _ in flows]
    for _ in range(6):
        for f, s, g in zip(flows, streams, got):
            g.append(f.run(stream=s))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for r in g for a, b in zip(r, w))
