"""Shared-prefix attention against a plain 64-bit implementation: every pair of
element types, head layouts, block sizes, groups nested or apart, single rows,
drafted tokens and prefill chunks, lengths from one key on.

Tolerance per output: with weights off by a relative w each, sum p v / sum p is
off by at most 2 w A, A = sum p |v| / sum p. w holds the half step of the
softmax weights' type (fp32 weights: the exponential's 2^-22), and the fp32
scores' own error: dot products of d terms, (d + 8) 2^-24 sum |q k| scale, and
the scaled score's rounding, 2^-22 |s|. Then one rounding to the output type."""
import ctypes
import math

import numpy as np
import pytest
import torch

from gpu_util import TORCH_DT

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


class Step:
    """seqs: (group, shared blocks, own keys, rows); a group's shared blocks are
    the first ones of one list per group, so deeper members extend shallower ones."""

    def __init__(self, seqs, heads, act="bf16", kv="bf16", block=16, seed=0, pool_extra=5, amp=1.0, **plan):
        from llm_engine_amd import kernels
        self.H, self.KH, self.d = heads
        self.bs = block
        self.dev = torch.device("cuda:0")
        rng = np.random.default_rng(seed)
        depth = {}
        for g, b, _, _ in seqs:
            depth[g] = max(depth.get(g, 0), b)
        own = [-(-k // block) for _, _, k, _ in seqs]
        used = sum(depth.values()) + sum(own)
        self.num_blocks = used + pool_extra
        ids = list(rng.permutation(self.num_blocks)[:used].astype(np.int32))
        shared = {g: [ids.pop() for _ in range(n)] for g, n in depth.items()}
        self.tables = [np.array(shared[g][:b] + [ids.pop() for _ in range(n)], dtype=np.int32)
                       for (g, b, _, _), n in zip(seqs, own)]
        self.keys = [b * block + k for _, b, k, _ in seqs]
        self.rows = [r for _, _, _, r in seqs]
        g = torch.Generator(device=self.dev)
        g.manual_seed(seed)
        n = sum(self.rows)

        def normal(*shape):
            return torch.randn(*shape, device=self.dev, generator=g)

        self.q = (amp * normal(n, self.H * self.d)).to(TORCH_DT[act])
        self.k = normal(self.num_blocks * block, self.KH * self.d).to(TORCH_DT[kv])
        self.v = normal(self.num_blocks * block, self.KH * self.d).to(TORCH_DT[kv])
        self.scale = 1.0 / math.sqrt(self.d)
        self.slices = [kernels.Slice(i, self.keys[i] - self.rows[i], self.rows[i], True, self.tables[i],
                                     np.zeros(self.keys[i], dtype=np.int32)) for i in range(len(seqs))]
        self.plan = kernels.PrefixPlan(self.slices, self.H, self.KH, self.d, block, TORCH_DT[kv], **plan).upload()

    def slots(self, i):
        return torch.from_numpy((self.tables[i].astype(np.int64)[:, None] * self.bs
                                 + np.arange(self.bs)).reshape(-1)[:self.keys[i]]).to(self.dev)

    def run(self, **kw):
        from llm_engine_amd import kernels
        return kernels.shared_prefix_attention(self.q, self.k, self.v, self.plan, self.scale, **kw)

    def want(self):
        """(outputs, tolerance) in 64 bits."""
        H, KH, d = self.H, self.KH, self.d
        G, outs, tols, r0 = H // KH, [], [], 0
        fp32 = self.q.dtype != self.k.dtype or self.k.dtype == torch.float32
        w0 = 2.0 ** -22 if fp32 else HALF_STEP[self.k.dtype]
        for i, (m, r) in enumerate(zip(self.keys, self.rows)):
            at = self.slots(i)
            k = self.k[at].double().reshape(m, KH, d).permute(1, 2, 0).contiguous()
            v = self.v[at].double().reshape(m, KH, d).permute(1, 0, 2).contiguous()
            q = self.q[r0:r0 + r].double().reshape(r, KH, G, d).permute(1, 2, 0, 3).reshape(KH, G * r, d)
            s = (q @ k) * self.scale
            big = ((q.abs() @ k.abs()) * abs(self.scale)).amax(-1)
            late = torch.arange(m, device=self.dev)[None] > torch.arange(m - r, m, device=self.dev)[:, None]
            late = late.repeat(G, 1)
            top = s.masked_fill(late, 0.0).abs().amax(-1)
            p = torch.softmax(s.masked_fill(late, -math.inf), dim=-1)
            o, a = p @ v, p @ v.abs()
            w = w0 + (d + 8) * 2.0 ** -24 * big + 2.0 ** -22 * top
            tol = 2 * w[..., None] * a + HALF_STEP[self.q.dtype] * (o.abs() + 2 * w[..., None] * a)

            def rows(x):
                return x.reshape(KH, G, r, d).permute(2, 0, 1, 3).reshape(r, H * d)

            outs.append(rows(o))
            tols.append(rows(tol) + 1e-7)
            r0 += r
        return torch.cat(outs), torch.cat(tols)

    def check(self, got=None):
        got = self.run() if got is None else got
        want, tol = self.want()
        over = (got.double() - want).abs() / tol
        assert not torch.isnan(got).any()
        assert float(over.max()) <= 1.0, f"{float(over.max())} times the tolerance"


QWEN, LLAMA, WIDE = (14, 2, 64), (32, 4, 64), (32, 8, 128)
BATCH = [(0, 20, k, 1) for k in (1, 15, 16, 17, 63, 64, 65, 130, 700, 3)]


@pytest.mark.parametrize("heads", [QWEN, LLAMA, WIDE, (4, 4, 64), (3, 3, 128), (8, 1, 128), (16, 2, 64)])
@pytest.mark.parametrize("kv", ["bf16", "f16", "f32"])
def test_one_group_of_decode_rows(gpu, heads, kv):
    s = Step(BATCH, heads, act=kv, kv=kv, seed=1)
    assert s.plan.groups == 1 and s.plan.saved_keys == 9 * 320
    s.check()


@pytest.mark.parametrize("act,kv", [(a, k) for a in ("f32", "bf16", "f16") for k in ("f32", "bf16", "f16") if a != k])
@pytest.mark.parametrize("heads", [QWEN, WIDE])
def test_mixed_types_are_fp32_products(gpu, heads, act, kv):
    Step(BATCH, heads, act=act, kv=kv, seed=2).check()


@pytest.mark.parametrize("block", [8, 16, 32, 64, 128, 512])
def test_block_sizes(gpu, block):
    seqs = [(0, -(-640 // block), k, 1) for k in (5, 100, 513, 70)] + [(1, 0, 900, 1), (1, 0, 1, 1)]
    Step(seqs, QWEN, block=block, seed=3).check()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_drafts_and_chunks_beside_decode_rows(gpu, kv):
    """Drafted tokens (2 to 8 rows), chunks that start right behind the shared
    blocks and later, in tiles of part of the columns and of several."""
    seqs = [(0, 12, 5, 5), (0, 12, 40, 2), (0, 12, 8, 8), (0, 12, 300, 200), (0, 12, 37, 37), (0, 12, 900, 1),
            (1, 9, 77, 3), (1, 9, 513, 512), (2, 0, 100, 100), (3, 0, 1, 1)]
    s = Step(seqs, QWEN, act=kv, kv=kv, seed=4)
    assert s.plan.groups == 2
    s.check()


def test_nested_prefixes(gpu):
    """Members that share more blocks with each other than with the rest: the
    cut that saves the most reads."""
    seqs = [(0, 8, 20, 1)] * 3 + [(0, 40, 30, 1)] * 4 + [(1, 3, 9, 1), (1, 4, 200, 1), (2, 100, 1, 1)]
    s = Step(seqs, LLAMA, seed=5)
    # 4 x 40 blocks (saved 120) against 7 x 8 (48); the three others share 8 among themselves (16)
    assert s.plan.groups >= 1 and s.plan.saved_keys >= 120 * 16
    s.check()


def test_nothing_shared_and_single_keys(gpu):
    s = Step([(i, 0, k, 1) for i, k in enumerate((1, 2, 63, 64, 65, 129, 2000, 16))], WIDE, seed=6)
    assert s.plan.groups == 0 and s.plan.saved_keys == 0
    s.check()
    s = Step([(0, 0, 1, 1)], QWEN, seed=7)
    assert s.plan.workspace_size() == 0
    s.check()


def test_full_blocks_only_are_shared(gpu):
    """A table that ends inside the shared blocks shares the whole ones before
    its row only, and a row that starts a block still sees itself."""
    s = Step([(0, 30, 1, 1), (0, 30, 2, 2), (0, 30, 50, 1)], QWEN, seed=8)
    s.check()
    # the same table for two sequences at different positions of it
    from llm_engine_amd import kernels
    s = Step([(0, 10, 16, 1), (0, 10, 16, 1)], QWEN, seed=9)
    s.keys, s.rows = [100, 176], [1, 1]
    s.tables[0] = s.tables[1]
    s.slices = [kernels.Slice(i, s.keys[i] - 1, 1, True, s.tables[i], np.zeros(176, np.int32)) for i in range(2)]
    s.plan = kernels.PrefixPlan(s.slices, *QWEN, 16, torch.bfloat16).upload()
    assert s.plan.groups == 1 and s.plan.saved_keys == 96
    s.check()


@pytest.mark.parametrize("part", [1, 64, 200, 100000])
def test_partitions_agree(gpu, part):
    seqs = [(0, 50, 333, 2), (0, 50, 1, 1), (0, 50, 64, 64), (1, 0, 1500, 1)]
    Step(seqs, QWEN, seed=10, partition_tokens=part).check()


@pytest.mark.parametrize("heads", [QWEN, WIDE])
def test_numbers_of_parts(gpu, heads):
    """Rows of 2 to 129 parts, one more or less than what a wave takes at a time."""
    own = [64 * n - 3 for n in (1, 2, 3, 6, 7, 8, 9, 14, 15, 16, 17, 30, 31, 32, 33, 47, 62, 63, 64, 65, 100, 128)]
    Step([(0, 8, k, 1) for k in own], heads, seed=20, partition_tokens=64, chunk_partition_tokens=128).check()


@pytest.mark.parametrize("tile", [32, 128])
@pytest.mark.parametrize("heads,kv", [(QWEN, "bf16"), (QWEN, "f32"), (WIDE, "f16"), (WIDE, "f32"), ((3, 3, 128), "bf16")])
def test_tile_widths(gpu, heads, kv, tile):
    """Tiles of at most 32 columns, or up to 128, asked for."""
    seqs = BATCH + [(0, 20, 90, 50), (1, 5, 64, 8), (1, 5, 3, 2), (2, 0, 140, 140)]
    Step(seqs, heads, act=kv, kv=kv, seed=21, chunk_q_tile=tile).check()


@pytest.mark.parametrize("heads,kv", [(QWEN, "bf16"), (WIDE, "f16"), (QWEN, "f32")])
def test_more_block_ids_than_lanes(gpu, heads, kv):
    """Items of several times 64 blocks, in wide tiles and in narrow ones."""
    seqs = [(0, 333, 5, 1)] * 9 + [(1, 0, 8 * 197 + 3, 1), (2, 0, 8 * 130, 40), (3, 64, 8, 8), (3, 64, 9, 9)]
    Step(seqs, heads, act=kv, kv=kv, block=8, seed=22, partition_tokens=100000, chunk_partition_tokens=100000,
         chunk_q_tile=128).check()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_nan_and_infinities_stay_with_their_rows(gpu, kv):
    """A q row, a key and a value of one sequence: the rows and heads that the
    formula makes NaN are, and no other output changes a bit."""
    s = Step(BATCH + [(0, 20, 60, 30)], QWEN, act=kv, kv=kv, seed=23)
    clean, G, d = s.run(), s.H // s.KH, s.d
    s.q[3, 2 * d + 1] = math.nan                                    # row 3, head 2
    s.k[s.slots(5)[s.keys[5] - 2], d + 4] = math.inf                # sequence 5, kv head 1
    s.v[s.slots(6)[s.keys[6] - 30], 9] = math.nan                   # sequence 6, kv head 0, dim 9
    s.q[8, 13 * d:] = -math.inf                                     # row 8, the last head
    got = s.run()
    want, _ = s.want()
    bad = torch.isnan(want)
    assert torch.equal(torch.isnan(got), bad)
    # where q's sign makes the infinite key score -inf, it drops out: no NaN,
    # and off by at most 2 w max|v| and one rounding (w as above, 1e-3 for the scores)
    drop = torch.zeros_like(bad)
    drop[5, G * d:] = ~bad[5, G * d:]
    assert bool(bad[5, G * d:].any()) and bool(drop.any())
    tol = (3 * HALF_STEP[s.q.dtype] + 1e-3) * float(s.v.float().nan_to_num().abs().max())
    assert float((got.double() - want)[drop].abs().max()) <= tol
    heads = (bad | drop).reshape(-1, s.H, d).any(-1).nonzero().tolist()
    assert heads == [[3, 2]] + [[5, h] for h in range(G, s.H)] + [[6, h] for h in range(G)] + [[8, 13]]
    assert torch.equal(got[~(bad | drop)], clean[~(bad | drop)])


@pytest.mark.parametrize("heads,n", [(LLAMA, 141), (WIDE, 75), ((3, 3, 128), 181), ((40, 5, 64), 109)])
@pytest.mark.parametrize("act,kv", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32")])
def test_many_short_sequences(gpu, heads, n, act, kv):
    """More workgroups than the chip holds: items of up to 32 keys take a wave
    each; drafts, keys from one on, and rows with nothing shared among them."""
    seqs = [(0, 12, 1 + i % 45, 1 + min(i % 45, i % 4)) for i in range(n)] + [(1 + i, 0, 1 + i, 1) for i in range(7)]
    s = Step(seqs, heads, act=act, kv=kv, seed=24)
    assert 0 < s.plan.plan.n_solo < s.plan.plan.n_items
    s.check()


@pytest.mark.parametrize("act,kv", [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")])
def test_very_many_short_sequences(gpu, act, kv):
    """Twice the workgroups that the chip holds: items of up to 64 keys take a wave."""
    s = Step([(0, 6, 1 + i % 80, 1) for i in range(170)], WIDE, act=act, kv=kv, seed=25)
    assert s.plan.plan.n_solo > 100
    s.check()


@pytest.mark.parametrize("heads", [LLAMA, (3, 3, 128)])
def test_nothing_but_short_sequences(gpu, heads):
    """Every item takes a wave; the last workgroup's waves are not all needed."""
    s = Step([(i, 0, 1 + i % 64, 1 + min(i % 64, i % 3)) for i in range(701)], heads, seed=26)
    assert s.plan.plan.n_solo == s.plan.plan.n_items == 701 and s.plan.workspace_size() == 0
    s.check()


@pytest.mark.parametrize("kv", ["bf16", "f16", "f32"])
def test_dead_cache_rows_are_not_read(gpu, kv):
    """NaN in every cache row that no sequence has computed (the rest of the last
    blocks, unused blocks)."""
    s = Step(BATCH + [(1, 0, 70, 30)], QWEN, act=kv, kv=kv, seed=11)
    live = torch.zeros(s.k.shape[0], dtype=torch.bool, device=s.dev)
    for i in range(len(s.keys)):
        live[s.slots(i)] = True
    s.k[~live] = math.nan
    s.v[~live] = math.nan
    s.check()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_large_scores(gpu, kv):
    """Scores in the hundreds: one key takes nearly everything, and running
    maxima move."""
    Step(BATCH, QWEN, act=kv, kv=kv, seed=12, amp=60.0).check()


@pytest.mark.parametrize("scale", [-0.125, 0.0])
def test_negative_and_zero_scale(gpu, scale):
    s = Step(BATCH, QWEN, seed=13)
    s.scale = scale
    s.check()


def test_blocks_outside_the_cache_read_as_zeros(gpu):
    s = Step([(0, 6, 40, 1), (0, 6, 90, 1)], QWEN, seed=14)
    s.tables[0][7], s.tables[1][8] = s.num_blocks + 3, -2
    from llm_engine_amd import kernels
    for i in range(2):
        s.slices[i].blocks = s.tables[i]
    s.plan = kernels.PrefixPlan(s.slices, *QWEN, 16, torch.bfloat16).upload()
    got = s.run()
    # the same step with those blocks in the cache, all zero
    s.k, s.v = (torch.cat([t, torch.zeros(16, t.shape[1], device=s.dev, dtype=t.dtype)]) for t in (s.k, s.v))
    s.tables[0][7] = s.tables[1][8] = s.num_blocks
    s.check(got)


def test_offsets_beyond_32_bits(gpu):
    """A cache of more than 2^32 bytes, the sequences' blocks at its end."""
    s = Step([(0, 20, 50, 1), (0, 20, 300, 2)], WIDE, seed=15)
    blocks = (5 << 30) // (16 * 8 * 128 * 2)
    k, v = (torch.empty(blocks * 16, 8 * 128, device=s.dev, dtype=torch.bfloat16) for _ in range(2))
    k[-s.k.shape[0]:], v[-s.k.shape[0]:] = s.k, s.v
    shift = blocks - s.num_blocks
    from llm_engine_amd import kernels
    s.tables = [t + shift for t in s.tables]
    for i in range(2):
        s.slices[i].blocks = s.tables[i]
    s.k, s.v = k, v
    s.plan = kernels.PrefixPlan(s.slices, *WIDE, 16, torch.bfloat16).upload()
    s.check()


def test_same_result_as_ragged_attention(gpu):
    """The two entry points on one step: within the sum of what each may be off."""
    from llm_engine_amd import kernels
    s = Step(BATCH + [(0, 20, 70, 40)], LLAMA, seed=16)
    plan = kernels.Plan(s.slices, *LLAMA, 16, torch.bfloat16).upload()
    a, b = s.run(), kernels.ragged_paged_attention(s.q, s.k, s.v, plan, s.scale)
    # the ragged kernels round scale * q to bf16 too: 2^-8 of every score
    want, tol = s.want()
    assert float(((a.double() - b.double()).abs() / (2 * tol + 0.05)).max()) <= 1.0


def test_other_stream_shared_workspace_and_graph(gpu):
    """Two steps through one workspace, on a stream of their own, replayed from
    a graph with other work between; outputs past the last row stay."""
    from llm_engine_amd import kernels
    a, b = Step(BATCH, QWEN, seed=17), Step([(0, 70, 200, 3), (0, 70, 5, 1), (0, 70, 99, 1)], QWEN, seed=18)
    ws = torch.empty(max(a.plan.workspace_size(), b.plan.workspace_size()), dtype=torch.uint8, device=a.dev)
    outs = [torch.full((s.q.shape[0] + 3, s.q.shape[1]), 7.0, dtype=s.q.dtype, device=a.dev) for s in (a, b)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def both():
        for s, o in zip((a, b), outs):
            s.run(out=o[:s.q.shape[0]], workspace=ws, stream=stream)

    both()
    stream.synchronize()
    first = [o.clone() for o in outs]
    a.check(outs[0][:-3])
    b.check(outs[1][:-3])
    assert all(bool((o[-3:] == 7).all()) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        both()
    for _ in range(3):
        for o in outs:
            o.fill_(7.0)
        ws.fill_(255)  # NaN patterns: nothing of an earlier launch is used
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, f) for o, f in zip(outs, first))
        torch.mm(torch.ones(64, 64, device=a.dev), torch.ones(64, 64, device=a.dev))


def test_launch_refusals(gpu):
    from llm_engine_amd import _lib, kernels
    s = Step(BATCH, QWEN, seed=19)
    with pytest.raises(ValueError):
        kernels.shared_prefix_attention(s.q[:-1], s.k, s.v, s.plan, 1.0)
    with pytest.raises(ValueError):
        kernels.shared_prefix_attention(s.q, s.k[:-1], s.v[:-1], s.plan, 1.0)
    with pytest.raises(_lib.LeError):
        kernels.shared_prefix_attention(s.q, s.k.float(), s.v.float(), s.plan, 1.0)  # planned for another type
    with pytest.raises(_lib.LeError):
        kernels.shared_prefix_attention(s.q, s.k, s.v, s.plan, math.nan)
    odd = torch.empty(s.q.numel() + 1, dtype=s.q.dtype, device=s.dev)[1:].view_as(s.q)
    with pytest.raises(_lib.LeError):
        kernels.shared_prefix_attention(odd, s.k, s.v, s.plan, s.scale)  # 2-byte aligned
    L, nul = _lib.load(), ctypes.c_void_p(0)
    st = L.le_shared_prefix_attention(s.q.data_ptr(), _lib.LE_BF16, s.k.data_ptr(), s.v.data_ptr(), _lib.LE_BF16,
                                      s.num_blocks, ctypes.byref(s.plan.plan), 0.125, s.q.data_ptr(), nul, 0, nul)
    assert st == _lib.LE_ENOSPACE
