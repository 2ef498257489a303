"""Host checks of the shared-prefix packer (le_prefix_plan_step) and of the
argument checks of the three operators around it (no GPU needed): every (row,
visible key) is in exactly one work item, with the right block id; parts and
records are numbered without gaps; shared blocks are read once."""
import ctypes

import numpy as np
import pytest
import torch

from llm_engine_amd import _lib, kernels

def pack(seqs, heads=(14, 2, 64), block=16, kv=torch.bfloat16, **kw):
    """seqs: (table, start, rows)."""
    slices = [kernels.Slice(i, a, r, True, np.array(t, dtype=np.int32), np.zeros(a + r, dtype=np.int32))
              for i, (t, a, r) in enumerate(seqs)]
    return kernels.PrefixPlan(slices, *heads, block, kv, device="cpu", pin=False, **kw)


def arrays(plan):
    P, b = plan.plan, plan.host.numpy()

    def at(off, n):
        return b[off:off + 4 * n].view(np.int32)

    items = at(P.off_items, 8 * P.n_items).reshape(-1, 8)
    rows = at(P.off_rows, 4 * P.n_items * P.rows_stride).reshape(P.n_items, -1, 4)
    listed = at(P.off_item_ids, P.n_items * P.ids_stride).reshape(P.n_items, -1)
    return (items, rows, listed, at(P.off_ids, int((P.off_part0 - P.off_ids) // 4)), at(P.off_part0, P.n_tokens),
            at(P.off_row_parts, P.n_tokens))


def check(seqs, heads=(14, 2, 64), block=16, **kw):
    plan = pack(seqs, heads, block, **kw)
    items, rows, listed, ids, part0, row_parts = arrays(plan)
    G = heads[0] // heads[1]
    tables = [t for t, _, r in seqs for _ in range(r)]
    positions = [a + j for _, a, r in seqs for j in range(r)]
    seen = [np.zeros(p + 1, dtype=int) for p in positions]
    parts = [[] for _ in positions]
    for i, (n, ido, kb, ke, part, causal, _, _) in enumerate(items):
        assert 0 < n * G <= 128 and 0 <= kb < ke and kb % block == 0
        for t, pos, first, _ in rows[i, :n]:
            assert pos == positions[t] and first == part0[t]
            e = min(ke, pos + 1)
            assert causal or ke <= pos + 1
            if e > kb:
                seen[t][kb:e] += 1
            for b in range(kb // block, (ke - 1) // block + 1):
                assert ids[ido + b - kb // block] == tables[t][b]
                if b - kb // block < 64:
                    assert listed[i, b - kb // block] == tables[t][b]
            parts[t].append(int(part))
        assert (rows[i, n:, 0] == rows[i, n - 1, 0]).all()  # padded with a row that exists
    assert all((s == 1).all() for s in seen)
    used = 0
    for t, p in enumerate(parts):
        assert row_parts[t] == len(p)
        if len(p) == 1:
            assert p == [-1]
        else:
            assert sorted(p) == list(range(len(p))) and part0[t] == used
            used += len(p)
    assert plan.plan.n_parts == used
    return plan


def test_groups_and_saved_reads():
    rng = np.random.default_rng(0)
    a, b = rng.permutation(1000)[:60], rng.permutation(1000)[:60]
    plan = check([(a[:30], 470, 1), (a, 900, 1), (list(a[:20]) + list(b[:9]), 450, 3)])
    # 20 blocks by three (40 saved) against 29 by two (29 saved)
    assert plan.groups == 1 and plan.saved_keys == 640
    plan = check([(a[:50], 799, 1), (a, 800, 1), (list(a[:20]) + list(b[:9]), 450, 3)])
    assert plan.groups == 1 and plan.saved_keys == 49 * 16
    plan = check([(a, 900, 1), (b, 900, 1), (a, 910, 1), (b, 700, 5)])
    assert plan.groups == 2 and plan.saved_keys == (56 + 43) * 16
    assert check([(a, 40, 1), (a, 47, 1)]).groups == 0  # 32 keys: not worth a pass
    assert check([(a, 64, 1), (a, 900, 1)]).saved_keys == 64


def test_a_slice_shares_only_what_is_before_it():
    a = np.arange(100)
    plan = check([(a, 0, 500), (a, 500, 1), (a, 80, 300), (a, 96, 1)])
    assert plan.groups == 1  # the prefill from 0 has nothing before it
    assert plan.saved_keys == max(2 * 80, 96)


@pytest.mark.parametrize("heads", [(14, 2, 64), (4, 4, 64), (8, 1, 128), (3, 1, 64)])
@pytest.mark.parametrize("block", [8, 16, 64, 512])
@pytest.mark.parametrize("part", [0, 1, 100, 4096])
def test_random_steps(heads, block, part):
    rng = np.random.default_rng(heads[0] * 1000 + block + part)
    for _ in range(6):
        base = [rng.integers(0, 1 << 20, 40) for _ in range(3)]
        seqs = []
        for _ in range(int(rng.integers(1, 25))):
            t = list(base[rng.integers(3)][:rng.integers(0, 41)]) + list(rng.integers(0, 1 << 20, rng.integers(1, 6)))
            n = int(rng.integers(1, min(len(t) * block, 900) + 1))
            rows = int(min(n, rng.choice([1, 1, 1, 2, 5, 64, 300])))
            seqs.append((t, n - rows, rows))
        check(seqs, heads, block, partition_tokens=part)


def test_deep_chain_of_prefixes():
    """Every table extends the one before: the tree of common beginnings is a chain."""
    a = np.arange(2000)
    plan = check([(a[:k + 1], 16 * k, 1) for k in range(0, 400, 4)])
    assert plan.groups == 1 and plan.saved_keys > 0


def test_many_sequences_behind_one_prompt():
    rng = np.random.default_rng(1)
    a = np.arange(256)
    plan = check([(np.concatenate([a, rng.integers(300, 9000, 30)]), 256 * 16 + int(k), 1)
                  for k in rng.integers(0, 400, 256)])
    assert plan.groups == 1 and plan.saved_keys == 255 * 4096


def test_slices_of_one_sequence_use_its_first_table():
    t = np.arange(10, dtype=np.int32)
    s = [kernels.Slice(7, 0, 20, False, t, np.zeros(60, np.int32)), kernels.Slice(7, 20, 4, True, t + 50, np.zeros(60, np.int32))]
    plan = kernels.PrefixPlan(s, 14, 2, 64, 16, torch.bfloat16, device="cpu", pin=False)
    ids = arrays(plan)[3]
    assert 50 not in ids and 51 not in ids


def test_empty_step():
    plan = pack([])
    assert plan.groups == 0 and plan.workspace_size() == 0 and plan.plan.n_tokens == 0
    nul = ctypes.c_void_p(0)
    L = _lib.load()
    assert L.le_prefix_plan_upload(ctypes.byref(plan.plan), nul, nul, nul) == _lib.LE_OK
    assert L.le_shared_prefix_attention(nul, 1, nul, nul, 1, 0, ctypes.byref(plan.plan), 1.0, nul, nul, 0, nul) == _lib.LE_OK


def test_packer_refusals():
    t = np.arange(4)
    for seqs, heads, block, status in (
            ([(t, 0, 0)], (14, 2, 64), 16, _lib.LE_EINVAL),       # no rows
            ([(t, -1, 1)], (14, 2, 64), 16, _lib.LE_EINVAL),
            ([(t, 64, 1)], (14, 2, 64), 16, _lib.LE_EINVAL),      # a position without a block
            ([(t, 2 ** 31 - 1, 1)], (14, 2, 64), 16, _lib.LE_EINVAL),
            ([(t, 5, 1)], (14, 3, 64), 16, _lib.LE_EINVAL),
            ([(t, 5, 1)], (18, 2, 64), 16, _lib.LE_EUNSUPPORTED),  # 9 heads a kv head
            ([(t, 5, 1)], (14, 2, 96), 16, _lib.LE_EUNSUPPORTED),
            ([(t, 5, 1)], (14, 2, 64), 12, _lib.LE_EUNSUPPORTED)):
        cfg = _lib.PlanConfig(*heads, block, _lib.LE_BF16, 0, 0, 0, 0, 0)
        b = np.ascontiguousarray(seqs[0][0], dtype=np.int32)
        s = (_lib.StepSlice * 1)(_lib.StepSlice(0, seqs[0][1], seqs[0][2], 1, b.size, b.ctypes.data, None))
        plan = _lib.PrefixStepPlan()
        assert _lib.load().le_prefix_plan_step(s, 1, ctypes.byref(cfg), None, 0, ctypes.byref(plan)) == status, seqs
    for field, value in (("flags", 4), ("table_capacity", 8), ("kv_dtype", 9), ("partition_tokens", -1),
                         ("chunk_q_tile", 16), ("chunk_partition_tokens", -1)):
        cfg = _lib.PlanConfig(14, 2, 64, 16, _lib.LE_BF16, 0, 0, 0, 0, 0)
        setattr(cfg, field, value)
        b = np.arange(4, dtype=np.int32)
        s = (_lib.StepSlice * 1)(_lib.StepSlice(0, 5, 1, 1, 4, b.ctypes.data, None))
        plan = _lib.PrefixStepPlan()
        assert _lib.load().le_prefix_plan_step(s, 1, ctypes.byref(cfg), None, 0, ctypes.byref(plan)) == _lib.LE_EINVAL
    with pytest.raises(_lib.LeError):
        pack([(t, 64, 1)])


def test_plans_larger_than_the_first_buffer():
    plan = pack([(np.arange(100_000), 800_000 - 1, 1)], block=8)  # 400 KB of ids
    assert plan.plan.bytes > 400_000 and plan.host.numel() >= plan.plan.bytes
    assert (arrays(plan)[3][:100_000] == np.arange(100_000)).all()


@pytest.mark.parametrize("differ", [0, 63, 64, 65, 127, 128, 190])
def test_common_beginnings_of_any_length(differ):
    """Two tables of 200 ids that differ at one place share what is before it."""
    a, b = np.arange(200), np.arange(200)
    b[differ] = 1000
    plan = check([(a, 1600 - 1, 1), (b, 1600 - 1, 1)], block=8)
    assert plan.saved_keys == (8 * differ if 8 * differ >= 64 else 0)


@pytest.mark.parametrize("seed", range(12))
def test_random_steps_in_asked_tiles(seed):
    rng = np.random.default_rng(100 + seed)
    tables = [rng.integers(0, 500, 60) for _ in range(3)]
    seqs = []
    for _ in range(int(rng.integers(1, 30))):
        depth, own = int(rng.integers(0, 50)), int(rng.integers(1, 40))
        table = np.concatenate([tables[rng.integers(0, 3)][:depth], rng.integers(500, 900, own)])
        rows = int(rng.integers(1, 1 + min(60, 16 * len(table))))
        seqs.append((table, 16 * len(table) - rows - int(rng.integers(0, min(15, 16 * len(table) - rows) + 1)), rows))
    heads = [(14, 2, 64), (32, 8, 128), (8, 1, 64), (5, 5, 64)][seed % 4]
    tile = 32 if seed % 2 else 128
    plan = check(seqs, heads, chunk_q_tile=tile, partition_tokens=int(rng.integers(0, 300)),
                 chunk_partition_tokens=int(rng.integers(0, 900)))
    assert (arrays(plan)[0][:, 0] * (heads[0] // heads[1]) <= tile).all()


@pytest.mark.parametrize("n,heads,kv,solo", [(40, (32, 4, 64), torch.bfloat16, False), (150, (32, 4, 64), torch.bfloat16, True),
                                             (40, (32, 8, 128), torch.float32, True), (40, (32, 8, 128), torch.bfloat16, False)])
def test_short_items_of_a_full_step_take_a_wave(n, heads, kv, solo):
    """The last items of the list, of at most 32 keys and columns."""
    seqs = [(np.concatenate([np.arange(20), 100 + 5 * i + np.arange(5)]), 320 + i % 70, 1 + i % 3) for i in range(n)]
    plan = check(seqs, heads, kv=kv)
    items, P = arrays(plan)[0], plan.plan
    assert (P.n_solo > 0) == solo
    short = (items[:, 3] - items[:, 2] <= 32) & (items[:, 0] * (heads[0] // heads[1]) <= 32)
    assert P.n_solo == (int(short.sum()) if solo else 0) and short[P.n_items - P.n_solo:].all()


def test_attention_refusals_without_launch():
    plan = pack([(np.arange(30), 400, 1), (np.arange(30), 410, 1)])
    P, L = plan.plan, _lib.load()
    fake, odd, nul = ctypes.c_void_p(4096), ctypes.c_void_p(4098), ctypes.c_void_p(0)

    def call(q=fake, act=1, kv=1, blocks=64, scale=0.125, out=fake, ws=fake, n=1 << 30, dev=4096, cache=fake):
        P.dev = dev
        return L.le_shared_prefix_attention(q, act, cache, fake, kv, blocks, ctypes.byref(P), scale, out, ws, n, nul)

    assert call(dev=None) == _lib.LE_EINVAL
    assert call(q=nul) == _lib.LE_EINVAL and call(out=nul) == _lib.LE_EINVAL and call(cache=nul) == _lib.LE_EINVAL
    assert call(act=5) == _lib.LE_EINVAL and call(kv=0) == _lib.LE_EINVAL and call(blocks=0) == _lib.LE_EINVAL
    assert call(scale=float("nan")) == _lib.LE_EINVAL
    assert call(q=odd) == _lib.LE_EUNSUPPORTED and call(out=odd) == _lib.LE_EUNSUPPORTED
    assert call(ws=nul) == _lib.LE_ENOSPACE and call(n=plan.workspace_size() - 1) == _lib.LE_ENOSPACE
    assert call(ws=odd) == _lib.LE_EUNSUPPORTED
    assert L.le_shared_prefix_attention(fake, 1, fake, fake, 1, 1, None, 1.0, fake, fake, 0, nul) == _lib.LE_EINVAL


def test_blocks_past_32_bit_offsets_are_refused():
    plan = pack([(np.arange(30), 400, 1), (np.arange(30), 410, 1)])
    P, L, fake = plan.plan, _lib.load(), ctypes.c_void_p(4096)
    P.dev = 4096
    P.cfg.q_heads = P.cfg.kv_heads = 1 << 15
    P.cfg.head_dim, P.cfg.block_size = 128, 512  # 2^15 * 128 * 2 bytes * 512 = 4 GiB
    st = L.le_shared_prefix_attention(fake, 1, fake, fake, 1, 64, ctypes.byref(P), 1.0, fake, fake, 0, None)
    assert st == _lib.LE_EUNSUPPORTED


def test_overlapping_outputs_and_endless_sequences_are_refused():
    plan = pack([(np.arange(30), 400, 1), (np.arange(30), 410, 1)])
    P, L = plan.plan, _lib.load()
    P.dev = 4096
    rows = 2 * 14 * 64 * 2
    for out in (1 << 20, (1 << 20) + rows - 16, (1 << 20) - rows + 16):
        st = L.le_shared_prefix_attention(1 << 20, 1, 4096, 4096, 1, 64, ctypes.byref(P), 1.0, out, 1 << 24, 1 << 30, None)
        assert st == _lib.LE_EINVAL
    one = (_lib.StepSlice * 1)()
    block = np.zeros(1 << 22, dtype=np.int32)
    for start, want in ((2**31 - 2, _lib.LE_EUNSUPPORTED), (2**31 - 4096, _lib.LE_EUNSUPPORTED), (2**31 - 1, _lib.LE_EINVAL)):
        one[0] = _lib.StepSlice(0, start, 1, 1, block.size, block.ctypes.data, None)
        cfg = _lib.PlanConfig(14, 2, 64, 512, _lib.LE_BF16, 0, 0, 0, 0, 0)
        assert L.le_prefix_plan_step(one, 1, ctypes.byref(cfg), None, 0, ctypes.byref(_lib.PrefixStepPlan())) == want


def test_verify_refusals_without_launch():
    L = _lib.load()
    fake, odd, nul = ctypes.c_void_p(4096), ctypes.c_void_p(4104), ctypes.c_void_p(0)

    def call(logits=fake, dt=0, stride=100, vocab=100, probs=fake, pdt=0, pstride=100, cu=fake, tok=fake, au=fake,
             su=fake, seqs=2, drafts=3, most=2, out=fake, ws=fake, n=1 << 30):
        return L.le_verify_drafts(logits, dt, stride, vocab, probs, pdt, pstride, cu, tok, au, su, nul, seqs, drafts,
                                  most, out, fake, ws, n, nul)

    for kw in (dict(logits=nul), dict(cu=nul), dict(tok=nul), dict(au=nul), dict(su=nul), dict(out=nul), dict(dt=7),
               dict(pdt=7), dict(vocab=0), dict(stride=99), dict(pstride=99), dict(seqs=-1), dict(drafts=-1),
               dict(most=-1)):
        assert call(**kw) == _lib.LE_EINVAL, kw
    for kw in (dict(seqs=65536), dict(most=65535), dict(ws=odd), dict(vocab=2 ** 31 - 1, stride=2 ** 31, pstride=2 ** 31)):
        assert call(**kw) == _lib.LE_EUNSUPPORTED, kw
    need = L.le_verify_drafts_workspace_size(2, 3, 100)
    assert call(n=need - 1) == _lib.LE_ENOSPACE and call(ws=nul) == _lib.LE_ENOSPACE
    assert call(seqs=0) == _lib.LE_OK
    assert L.le_verify_drafts_workspace_size(0, 3, 100) == 0


def test_qk_norm_refusals_without_launch():
    L = _lib.load()
    fake, odd, nul = ctypes.c_void_p(4096), ctypes.c_void_p(4104), ctypes.c_void_p(0)

    def call(qkv=fake, dt=1, stride=18 * 64, bias=nul, qn=fake, eps=1e-6, pos=fake, max_pos=10, n=4, heads=(14, 2, 64),
             q=fake, kc=fake, cdt=1, slots=100):
        return L.le_qk_norm_rope_kv_cache_write(qkv, dt, stride, bias, qn, fake, eps, pos, fake, fake, fake, max_pos, n,
                                                *heads, q, kc, fake, cdt, slots, nul)

    for kw in (dict(qkv=nul), dict(qn=nul), dict(pos=nul), dict(q=nul), dict(kc=nul), dict(dt=3), dict(cdt=-1),
               dict(stride=18 * 64 - 8), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
               dict(max_pos=0), dict(n=-1), dict(heads=(0, 2, 64)), dict(heads=(14, 0, 64)), dict(slots=-1)):
        assert call(**kw) == _lib.LE_EINVAL, kw
    for kw in (dict(stride=18 * 64 + 4), dict(heads=(14, 2, 60)), dict(heads=(14, 2, 520), stride=18 * 520),
               dict(qkv=odd), dict(bias=odd), dict(q=odd), dict(kc=odd), dict(qn=odd)):
        assert call(**kw) == _lib.LE_EUNSUPPORTED, kw
    assert call(n=0) == _lib.LE_OK
