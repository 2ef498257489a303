"""verify_drafts against a plain float64 implementation: token for token.
Weights are fp32 (relative error about 1e-7 each, independent), sums and
comparisons fp64, so a random number decides otherwise only if it falls within
about 1e-7 of a border: the seeds below are fixed."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def target(x, t):
    """Probabilities of one row of logits (float64) at temperature t."""
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    p = np.zeros_like(x)
    if m == -np.inf:
        p[0] = 1
        return p
    if not t > 0:
        p[int(np.argmax(x))] = 1
        return p
    if m == np.inf:
        p = (x == m).astype(np.float64)
    else:
        p = np.exp((x - m) / t)
    return p / p.sum()


def sample(p, u):
    mass = np.cumsum(p)
    over = np.nonzero(mass > u * mass[-1])[0]
    return int(over[0]) if len(over) else int(np.nonzero(p)[0][-1])


def plain(logits, cu, tokens, au, su, max_drafts, probs, temps):
    V = logits.shape[1]
    out = np.full((len(cu) - 1, max_drafts + 1), -1, dtype=np.int32)
    acc = np.zeros(len(cu) - 1, dtype=np.int32)
    for s in range(len(cu) - 1):
        if cu[s] < 0 or cu[s + 1] < cu[s] or cu[s + 1] > len(tokens) or cu[s + 1] - cu[s] > max_drafts:
            acc[s] = -1
            continue
        t = 1.0 if temps is None else float(temps[s])
        for j in range(cu[s], cu[s + 1] + 1):
            p = target(logits[j + s], t)
            if j < cu[s + 1]:
                x = int(tokens[j])
                inside = 0 <= x < V
                q = None if probs is None else probs[j]
                if inside and float(au[j]) * (1.0 if q is None else q[x]) < p[x]:
                    out[s, acc[s]] = x
                    acc[s] += 1
                    continue
                r = p.copy()
                if q is not None:
                    with np.errstate(invalid="ignore"):
                        r = np.fmax(p - q, 0.0)
                elif inside:
                    r[x] = 0.0
                p = r if t > 0 and r.sum() > 0 else p
            out[s, acc[s]] = sample(p, float(su[s]))
            break
    return out, acc


class Case:
    def __init__(self, drafts, vocab, logits="f32", probs="f32", temps=None, seed=0, spread=4.0, stride=0):
        self.dev = torch.device("cuda:0")
        g = torch.Generator(device=self.dev)
        g.manual_seed(seed)
        self.n = np.array(drafts, dtype=np.int64)
        self.cu = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        S, N = len(drafts), int(self.n.sum())
        self.max_drafts = int(self.n.max())
        seq = torch.from_numpy(np.repeat(np.arange(S), self.n)).to(self.dev)
        full = (spread * torch.randn(N + S, vocab + stride, device=self.dev, generator=g)).to(DT[logits])
        self.logits = full[:, :vocab]
        self.temps = None if temps is None else torch.tensor(temps, device=self.dev, dtype=torch.float32)
        near = self.logits[torch.arange(N, device=self.dev) + seq].float() + torch.randn(N, vocab, device=self.dev, generator=g)
        q = torch.softmax(near, -1)
        self.tokens = (torch.multinomial(q, 1, generator=g)[:, 0] if N else torch.zeros(0, device=self.dev)).to(torch.int32)
        self.probs = None if probs is None else q.to(DT[probs])
        self.au = torch.rand(N, device=self.dev, generator=g)
        self.su = torch.rand(S, device=self.dev, generator=g)

    def want(self):
        def n(t):
            return None if t is None else t.double().cpu().numpy()
        return plain(n(self.logits), self.cu.tolist(), self.tokens.tolist(), n(self.au), n(self.su), self.max_drafts,
                     n(self.probs), n(self.temps))

    def run(self, **kw):
        from llm_engine_amd import kernels
        return kernels.verify_drafts(self.logits, torch.from_numpy(self.cu).to(self.dev), self.tokens, self.au, self.su,
                                     self.max_drafts, draft_probs=self.probs, temperature=self.temps, **kw)

    def check(self, got=None):
        out, acc = self.run() if got is None else got
        want, count = self.want()
        assert np.array_equal(acc.cpu().numpy(), count), (acc.tolist(), count.tolist())
        assert np.array_equal(out.cpu().numpy(), want), (out.tolist(), want.tolist())
        return count


@pytest.mark.parametrize("vocab", [1, 7, 511, 512, 513, 2047, 2048, 2049, 32000, 65537, 151936])
def test_vocabularies(gpu, vocab):
    c = Case([4, 1, 3, 0, 5], vocab, temps=[1.0, 0.7, 0.0, 1.3, 0.2], seed=vocab)
    c.check()


@pytest.mark.parametrize("logits", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("probs", ["f32", "bf16", "f16", None])
def test_types(gpu, logits, probs):
    acc = Case([3] * 24, 5003, logits, probs, temps=list(np.linspace(0.3, 1.5, 24)), seed=3).check()
    assert 0 < acc.mean() < 3  # both outcomes


@pytest.mark.parametrize("stride", [0, 1, 3, 8])
@pytest.mark.parametrize("logits", ["f32", "bf16"])
def test_row_strides(gpu, logits, stride):
    c = Case([2, 4, 1], 3001, logits, "bf16", seed=stride + 5, stride=stride)
    c.check()


def test_sampling_only(gpu):
    Case([0] * 9, 40001, temps=[1.0] * 4 + [0.0] * 2 + [0.5] * 3, seed=6).check()


def test_all_accepted_and_all_rejected(gpu):
    c = Case([5, 5], 999, seed=7)
    c.au.zero_()
    assert (c.check() == 5).all()
    c.au.fill_(1.0 - 2.0 ** -24)
    c.probs.fill_(1.0)
    assert (c.check() == 0).all()


def test_greedy_ties_and_drafts(gpu):
    c = Case([2, 2, 2], 6000, "bf16", temps=[0.0, -1.0, math.nan], seed=8)
    rows = c.logits
    rows[:, [17, 400, 5999]] = 60.0                # tie: the lowest index
    c.tokens[:] = torch.tensor([17, 400, 17, 17, 5999, 17], dtype=torch.int32)
    acc = c.check()
    assert acc.tolist() == [1, 2, 0]


def test_masked_and_infinite_logits(gpu):
    c = Case([1] * 8, 4100, "f32", None, temps=[1.0] * 7 + [0.0], seed=9)
    x = c.logits
    x[0:2] = -math.inf                             # nothing left: token 0
    x[2:4] = -3.0e38                               # the type's lowest value: all alike
    x[4, 1::2] = -math.inf                         # a mask
    x[4:6, ::7] = math.nan
    x[6:8, [33, 2222]] = math.inf                  # share the mass
    x[8:10] = 3.0e38
    x[10:12, :] = -math.inf
    x[10:12, 4099] = -5.0                          # one token, the last
    x[12:14, 100:] = -math.inf
    x[14:16] = math.nan
    c.tokens[:] = torch.tensor([5, 7, 3, 2222, 9, 17, 99, 0], dtype=torch.int32)
    c.check()


def test_residual_without_mass_falls_back(gpu):
    """A draft rejected where its probabilities exceed the target's everywhere."""
    c = Case([1, 1], 3000, seed=10)
    c.probs.fill_(1.0)
    c.au.fill_(0.999)
    c.check()


@pytest.mark.parametrize("vocab", [5, 8192, 8193, 30011])
def test_rejected_lookup_drafts(gpu, vocab):
    """Drafts without probabilities that are rejected: at a piece's ends, with
    nearly all of the row's mass, alone in their piece, alone in the row (sampled
    after all), and with nothing of their own."""
    at = [0, vocab // 2, vocab - 1, min(8191, vocab - 1), min(8192, vocab - 1), vocab - 2, 3, 1]
    c = Case([1] * 8, vocab, "f32", None, seed=40 + vocab)
    c.tokens[:] = torch.tensor(at, dtype=torch.int32)
    c.au.fill_(1.0 - 2.0 ** -24)
    x = c.logits
    for i in range(3):
        x[2 * i, at[i]] = 30.0                     # e^30 against about vocab e^8 at most
    for i in (3, 4):                               # the piece's only token
        lo = at[i] // 8192 * 8192
        keep = x[2 * i, at[i]].clone()
        x[2 * i, lo:lo + 8192] = -math.inf
        x[2 * i, at[i]] = keep
    x[10] = -math.inf
    x[10, at[5]] = 1.0
    x[12, at[6]] = -math.inf
    x[14, at[7]] = math.nan
    acc = c.check().tolist()
    assert acc[6] == acc[7] == 0


def test_bad_tokens_offsets_and_random_numbers(gpu):
    c = Case([2, 3, 1, 2], 2500, seed=11)
    c.tokens[0], c.tokens[3] = -1, 2500            # no such tokens: rejected
    c.check()
    c = Case([2, 3, 1, 2], 2500, seed=12)
    c.cu = np.array([0, 2, 1, 6, 9], dtype=np.int32)  # decreasing, too many, past the end
    c.check()
    c = Case([1] * 4, 2500, seed=13)
    c.su[:] = torch.tensor([1.0, 2.0, 0.0, math.nan])
    c.au[:] = torch.tensor([1.0, math.nan, 0.0, 0.5])
    out, acc = c.run()
    want, count = c.want()
    assert acc.cpu().tolist() == count.tolist()
    # at 1 or NaN: the last token with any mass
    assert out.cpu()[2].tolist() == want[2].tolist()
    assert all(0 <= int(t) < 2500 for t in out.cpu()[torch.arange(4), acc.cpu().long()])


@pytest.mark.parametrize("t", [1e-30, 1e-4, 100.0, math.inf])
def test_extreme_temperatures(gpu, t):
    Case([2] * 6, 3333, "f16", None, temps=[t] * 6, seed=14).check()


def test_many_sequences_and_wide_gaps(gpu):
    rng = np.random.default_rng(15)
    Case(list(rng.integers(0, 9, 300)), 1200, seed=15).check()
    c = Case([1, 0], 1500, seed=16)
    c.max_drafts = 40                              # longer output rows than drafts
    c.check()


def test_stream_workspace_and_graph(gpu):
    from llm_engine_amd import kernels
    c = Case([3, 5, 0, 2], 50021, temps=[1.0, 0.5, 0.9, 0.0], seed=17)
    ws = torch.full((kernels.verify_drafts_workspace_size(4, 10, 50021),), 255, dtype=torch.uint8, device=c.dev)
    cu = torch.from_numpy(c.cu).to(c.dev)
    out, acc = torch.empty(4, 6, dtype=torch.int32, device=c.dev), torch.empty(4, dtype=torch.int32, device=c.dev)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def call():
        kernels.verify_drafts(c.logits, cu, c.tokens, c.au, c.su, 5, draft_probs=c.probs, temperature=c.temps, out=out,
                              n_accepted=acc, workspace=ws, stream=stream)

    call()
    stream.synchronize()
    c.check((out, acc))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for i in range(3):
        c.su.uniform_(generator=torch.Generator(device=c.dev).manual_seed(i))
        c.au.uniform_(generator=torch.Generator(device=c.dev).manual_seed(i + 9))
        out.fill_(77)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check((out, acc))


def test_distribution(gpu):
    """Accepted or resampled, the first token is distributed as the target says:
    40000 sequences over 5 tokens, within 5 standard deviations."""
    from llm_engine_amd import kernels
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(18)
    S, V = 40000, 5
    p = torch.tensor([0.4, 0.05, 0.3, 0.2, 0.05], device=dev)
    q = torch.tensor([0.1, 0.5, 0.1, 0.1, 0.2], device=dev)
    tokens = torch.multinomial(q.expand(S, V), 1, generator=g)[:, 0].to(torch.int32)
    out, _ = kernels.verify_drafts(p.log().expand(2 * S, V).contiguous(), torch.arange(S + 1, device=dev, dtype=torch.int32),
                                   tokens, torch.rand(S, device=dev, generator=g), torch.rand(S, device=dev, generator=g),
                                   1, draft_probs=q.expand(S, V).contiguous())
    share = torch.bincount(out[:, 0].long(), minlength=V).double().cpu() / S
    sd = (p.double().cpu() * (1 - p.double().cpu()) / S).sqrt()
    assert float(((share - p.double().cpu()).abs() / sd).max()) < 5


def test_refusals(gpu):
    from llm_engine_amd import _lib, kernels
    c = Case([2, 1], 300, seed=19)
    cu = torch.from_numpy(c.cu).to(c.dev)
    with pytest.raises(ValueError):
        kernels.verify_drafts(c.logits[:-1], cu, c.tokens, c.au, c.su, 2)
    with pytest.raises(ValueError):
        kernels.verify_drafts(c.logits, cu, c.tokens, c.au[:-1], c.su, 2)
    with pytest.raises(ValueError):
        kernels.verify_drafts(c.logits, cu, c.tokens, c.au, c.su, 2, draft_probs=c.probs[:, :-1])
    with pytest.raises(ValueError):
        kernels.verify_drafts(c.logits, cu.long(), c.tokens, c.au, c.su, 2)
    with pytest.raises(ValueError):  # one column for all
        kernels.verify_drafts(c.logits[:, :1].expand(5, 300), cu, c.tokens, c.au, c.su, 2)
    with pytest.raises(_lib.LeError):  # one row for all
        kernels.verify_drafts(c.logits[:1].expand(5, 300), cu, c.tokens, c.au, c.su, 2)
