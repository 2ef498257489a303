"""qk_norm_rope_store_kv against a plain 64-bit implementation.

Tolerance: the mean of squares of d terms is off by a relative (d / 8 + 16)
2^-24 at most, the norm by half of that and a few roundings, the rotation by
three roundings of its two products: (d / 8 + 24) 2^-24 (|x cos| + |y sin|).
Then one rounding to the stored type (fp16: subnormals, 2^-25)."""
import math

import numpy as np
import pytest
import torch

from gpu_util import TORCH_DT

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
EPS = 1e-6


class Case:
    def __init__(self, n, heads, act="bf16", kv="bf16", bias=False, stride=0, max_pos=512, seed=0, pool=None):
        self.n, (self.H, self.KH, self.d) = n, heads
        self.dev = torch.device("cuda:0")
        g = torch.Generator(device=self.dev)
        g.manual_seed(seed)

        def normal(*shape):
            return torch.randn(*shape, device=self.dev, generator=g)

        H, KH, d = heads
        width = (H + 2 * KH) * d
        pool = pool or (n + 15) // 16 * 16 + 32
        self.qkv = (1.7 * normal(n, width + stride)).to(TORCH_DT[act])[:, :width]
        self.bias = 0.5 * normal(width) if bias else None
        self.qw, self.kw = 1 + 0.3 * normal(d), 1 + 0.3 * normal(d)
        ang = torch.arange(max_pos, device=self.dev, dtype=torch.float64)[:, None] * 1e4 ** (
            -torch.arange(0, d, 2, device=self.dev, dtype=torch.float64) / d)
        self.cos, self.sin = ang.cos().float(), ang.sin().float()
        self.pos = torch.randint(0, max_pos, (n,), device=self.dev, generator=g, dtype=torch.int32)
        self.slots = torch.randperm(pool, device=self.dev, generator=g)[:n].to(torch.int32)
        self.k, self.v = (normal(pool, KH * d).to(TORCH_DT[kv]) for _ in range(2))
        self.eps = EPS

    def run(self, **kw):
        from llm_engine_amd import kernels
        return kernels.qk_norm_rope_store_kv(self.qkv, self.pos, self.slots, self.cos, self.sin, self.qw, self.kw,
                                             self.eps, self.H, self.KH, self.d, self.k, self.v, bias=self.bias, **kw)

    def check(self, run=None):
        H, KH, d = self.H, self.KH, self.d
        x = self.qkv.double()
        if self.bias is not None:
            x = x + self.bias.double()
        x = x.reshape(self.n, H + 2 * KH, d)
        w = torch.cat([self.qw.expand(H, d), self.kw.expand(KH, d)]).double()
        y = x[:, :H + KH]
        y = y / (y.square().mean(-1, keepdim=True) + self.eps).sqrt() * w
        here = (self.pos >= 0) & (self.pos < self.cos.shape[0])
        at = torch.where(here, self.pos, 0).long()
        cos, sin = self.cos[at].double()[:, None], self.sin[at].double()[:, None]
        a, b = y.chunk(2, dim=-1)
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        size = torch.cat([(a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()], -1)
        rot = torch.where(here[:, None, None], rot, 0.0)
        err = (d / 8 + 24) * 2.0 ** -24 * size
        rows = self.slots.long()
        stored = here & (rows >= 0) & (rows < self.k.shape[0])
        k0, v0 = self.k.clone(), self.v.clone()
        q = (run or self.run)()
        tol = err + HALF_STEP[q.dtype] * (rot.abs() + err) + 2.0 ** -25
        assert bool(((q.double().reshape(self.n, H, d) - rot[:, :H]).abs() <= tol[:, :H]).all())
        tol = err + HALF_STEP[self.k.dtype] * (rot.abs() + err) + 2.0 ** -25
        got = self.k[rows[stored]].double().reshape(-1, KH, d)
        assert bool(((got - rot[stored, H:]).abs() <= tol[stored, H:]).all())
        want = x[stored, H + KH:].reshape(-1, KH * d)
        tol = 2.0 ** -24 * want.abs() + HALF_STEP[self.v.dtype] * want.abs() * (1 + 2.0 ** -20) + 2.0 ** -25
        assert bool(((self.v[rows[stored]].double() - want).abs() <= tol).all())
        kept = torch.ones(self.k.shape[0], dtype=torch.bool, device=self.dev)
        kept[rows[stored]] = False
        assert torch.equal(self.k[kept], k0[kept]) and torch.equal(self.v[kept], v0[kept])
        return q


@pytest.mark.parametrize("act,kv", [(a, k) for a in ("f32", "bf16", "f16") for k in ("f32", "bf16", "f16")])
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128)])
def test_types(gpu, heads, act, kv):
    Case(37, heads, act, kv, bias=True, seed=1).check()


@pytest.mark.parametrize("d", [8, 16, 24, 40, 64, 72, 80, 96, 112, 128, 192, 256, 512])
def test_head_dims(gpu, d):
    Case(9, (3, 1, d), "bf16", "bf16", seed=d).check()
    Case(5, (2, 2, d), "f32", "f32", bias=True, seed=d + 1).check()


@pytest.mark.parametrize("n", [1, 2, 63, 64, 257, 4097])
@pytest.mark.parametrize("heads", [(14, 2, 64), (1, 1, 64), (40, 8, 128)])
def test_row_counts(gpu, n, heads):
    Case(n, heads, seed=n).check()


@pytest.mark.parametrize("stride", [8, 64, 1000])
def test_row_strides(gpu, stride):
    Case(33, (14, 2, 64), "f16", "bf16", stride=stride, seed=stride).check()


def test_padding_and_positions_outside(gpu):
    c = Case(50, (14, 2, 64), seed=5)
    c.slots[::7] = -1
    c.slots[3] = c.k.shape[0]
    c.slots[4] = 2 ** 31 - 1
    c.pos[5], c.pos[6], c.pos[8] = -1, c.cos.shape[0], 2 ** 31 - 1
    q = c.check()
    assert bool((q[[5, 6, 8]] == 0).all())


def test_zero_small_and_huge_rows(gpu):
    for act in ("f32", "bf16"):
        c = Case(6, (4, 2, 128), act, act, seed=6)
        c.qkv[0] = 0
        c.qkv[1] *= 1e-12
        c.qkv[2] *= 1e10
        c.qkv[3, ::2] = 0
        c.check()


def test_nothing_to_do(gpu):
    c = Case(1, (2, 1, 64), seed=7)
    from llm_engine_amd import kernels
    k0 = c.k.clone()
    q = kernels.qk_norm_rope_store_kv(c.qkv[:0], c.pos[:0], c.slots[:0], c.cos, c.sin, c.qw, c.kw, EPS, 2, 1, 64, c.k,
                                      c.v)
    assert q.shape == (0, 128) and torch.equal(c.k, k0)


def test_slots_beyond_32_bits(gpu):
    """A K cache of more than 2^32 bytes: the last slots."""
    c = Case(20, (10, 8, 128), seed=8)
    pool = (5 << 30) // (8 * 128 * 2)
    c.k, c.v = (torch.zeros(pool, 8 * 128, device=c.dev, dtype=torch.bfloat16) for _ in range(2))
    c.slots = (pool - 1 - torch.arange(20, device=c.dev)).to(torch.int32)
    c.check()


def test_stream_and_graph(gpu):
    c = Case(65, (14, 2, 64), seed=9)
    out = torch.empty(65, 14 * 64, dtype=torch.bfloat16, device=c.dev)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def run():
        r = c.run(q_out=out, stream=stream)
        stream.synchronize()
        return r

    c.check(run)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        c.run(q_out=out, stream=stream)
    for i in range(3):
        c.qkv.copy_(torch.randn(c.qkv.shape, device=c.dev, generator=torch.Generator(device=c.dev).manual_seed(i)))
        out.zero_()

        def replay():
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            return out

        c.check(replay)


def test_refusals(gpu):
    from llm_engine_amd import _lib, kernels
    c = Case(4, (14, 2, 64), seed=10)
    args = [c.qkv, c.pos, c.slots, c.cos, c.sin, c.qw, c.kw, EPS, 14, 2, 64, c.k, c.v]

    def but(i, x):
        return args[:i] + [x] + args[i + 1:]

    for i, x in ((0, c.qkv[:, :-1]), (1, c.pos.long()), (2, c.slots[:3]), (3, c.cos[:, :-1]), (5, c.qw[:-1]),
                 (5, c.qw.double()), (11, c.k[:, :-1]), (12, c.v.float())):
        with pytest.raises(ValueError):
            kernels.qk_norm_rope_store_kv(*but(i, x))
    for e in (-1.0, math.nan, math.inf):
        with pytest.raises(_lib.LeError):
            kernels.qk_norm_rope_store_kv(*but(7, e))
    wide = torch.zeros(4, 18 * 64 + 3, dtype=torch.bfloat16, device=c.dev)
    with pytest.raises(_lib.LeError):  # rows that are not whole 16-byte pieces
        kernels.qk_norm_rope_store_kv(*but(0, wide))
    with pytest.raises(_lib.LeError):  # one row for all tokens
        kernels.qk_norm_rope_store_kv(*but(0, c.qkv[:1].expand(4, -1)))
