"""CPU: what the attention-layer operators refuse before anything is launched, and the frequencies of rotated pairs."""
import ctypes as C
import math

import pytest
import torch

from vortex_b200 import _lib, attn_ops


def refused(fn, p, code, text):
    assert fn(C.byref(p), None) == code and text in _lib.last_error(), _lib.last_error()


def rotary(**kw):
    base = dict(q=16, k=16, q_out=16, k_out=16, positions=16, inv_freq=16, rot=64, B=1, L=3, Hq=2, Hk=1, D=64, io_dtype=1, scale=1.0)
    return _lib.RotaryParams(**{**base, **kw})


@pytest.mark.parametrize("bad,code,text", [
    (dict(io_dtype=7), -1, "dtype"), (dict(D=0), -1, "size"), (dict(L=-1), -1, "size"), (dict(D=513, rot=0), -2, "513"),
    (dict(rot=65), -1, "rotated"), (dict(rot=66), -1, "rotated"), (dict(rot=-2), -1, "rotated"), (dict(q=None), -1, "null"),
    (dict(k=None), -1, "null"), (dict(q_out=None), -1, "null"), (dict(positions=None), -1, "null"), (dict(inv_freq=None), -1, "null"),
    (dict(q_weight=16, q_weight_dtype=9), -1, "weight"), (dict(Hq=1 << 20), -2, "heads")])
def test_rotary_refusals(bad, code, text):
    lib = _lib.lib()
    refused(lib.vtx_qk_norm_rotary_fwd, rotary(**bad), code, text)
    if "q_out" not in bad:
        f = rotary(**bad)
        refused(lib.vtx_qk_norm_rotary_bwd, _lib.RotaryBwdParams(fwd=f, dq_out=16, dk_out=16), code, text)
        refused(lib.vtx_rotary_append, _lib.RotaryAppendParams(rot=f, v=16, k_pages=16, v_pages=16, block_table=16, table_width=2, num_seqs=3,
                                                               num_pages=4, page_size=16), code, text)


def test_rotary_of_nothing_needs_no_pointers():
    for kw in (dict(L=0), dict(B=0), dict(Hq=0, Hk=0)):
        p = rotary(q=None, k=None, q_out=None, k_out=None, **kw)
        assert _lib.lib().vtx_qk_norm_rotary_fwd(C.byref(p), None) == 0


def test_rotary_backward_refusals():
    lib = _lib.lib()
    f = rotary(q_weight=16, q_weight_dtype=0)
    assert lib.vtx_qk_norm_rotary_bwd_scratch_bytes(C.byref(f)) % (2 * 64 * 4) == 0 < lib.vtx_qk_norm_rotary_bwd_scratch_bytes(C.byref(f))
    assert lib.vtx_qk_norm_rotary_bwd_scratch_bytes(C.byref(rotary())) == 0
    mk = lambda **kw: _lib.RotaryBwdParams(**{**dict(fwd=f, dq_out=16, dk_out=16, dq_weight=16, scratch=16), **kw})  # noqa: E731
    refused(lib.vtx_qk_norm_rotary_bwd, mk(scratch=None), -1, "scratch")
    refused(lib.vtx_qk_norm_rotary_bwd, mk(dq_weight=None), -1, "weight gradient")
    refused(lib.vtx_qk_norm_rotary_bwd, mk(dk_out=None), -1, "null")
    assert lib.vtx_qk_norm_rotary_bwd(None, None) == lib.vtx_qk_norm_rotary_fwd(None, None) == lib.vtx_rotary_append(None, None) == -1


@pytest.mark.parametrize("bad,text", [(dict(page_size=0), "cache sizes"), (dict(num_pages=-1), "cache sizes"), (dict(v=None), "null"),
                                      (dict(k_pages=None), "null"), (dict(block_table=None), "null"), (dict(num_seqs=2), "rows of the block table")])
def test_append_refusals(bad, text):
    base = dict(rot=rotary(), v=16, k_pages=16, v_pages=16, block_table=16, table_width=2, num_seqs=3, num_pages=4, page_size=16)
    refused(_lib.lib().vtx_rotary_append, _lib.RotaryAppendParams(**{**base, **bad}), -1, text)
    refused(_lib.lib().vtx_rotary_append, _lib.RotaryAppendParams(**{**base, "rot": rotary(Hk=0)}), -1, "key heads")


def decode(**kw):
    base = dict(q=16, k_pages=16, v_pages=16, block_table=16, table_width=8, seqlens=16, out=16, scratch=16, softmax_scale=1.0, B=2, Hq=8, Hk=2,
                D=128, num_pages=40, page_size=16, io_dtype=1, q_stride_b=1024, q_stride_h=128, k_stride_page=4096, k_stride_slot=256,
                k_stride_head=128, v_stride_page=4096, v_stride_slot=256, v_stride_head=128, out_stride_b=1024, out_stride_h=128)
    return _lib.PagedDecodeParams(**{**base, **kw})


@pytest.mark.parametrize("bad,code,text", [
    (dict(io_dtype=3), -1, "dtype"), (dict(B=-1), -1, "sizes"), (dict(Hk=0), -1, "sizes"), (dict(Hq=7), -1, "7 query heads for 2"),
    (dict(D=257), -2, "257"), (dict(D=0), -1, "sizes"), (dict(page_size=0), -1, "sizes"), (dict(window=-1), -1, "window"),
    (dict(B=1 << 24), -2, "sequences"), (dict(num_pages=2 ** 31), -2, "pages"), (dict(block_table=None, num_pages=1), -1, "no block table"),
    (dict(q=None), -1, "null"), (dict(k_pages=None), -1, "null"), (dict(seqlens=None), -1, "null"), (dict(out=None), -1, "null"),
    (dict(scratch=None), -1, "scratch"), (dict(scratch=24), -1, "scratch")])
def test_decode_attention_refusals(bad, code, text):
    refused(_lib.lib().vtx_paged_decode_attention, decode(**bad), code, text)


def test_decode_attention_scratch():
    """Grows with the blocks that a call can use, not with its batch; nothing is needed where there is nothing to do."""
    f = _lib.lib().vtx_paged_decode_scratch_bytes
    n = lambda **kw: f(C.byref(decode(**kw)))  # noqa: E731
    assert n(B=0) == 0 and n(Hq=7) == 0 and f(None) == 0
    assert 0 < n(B=1, table_width=1) < n(B=1, table_width=100) < n(B=64, table_width=512) == n(B=4096, table_width=1 << 16)
    assert n(B=64, table_width=512) < 8 << 20
    assert n(B=64, table_width=2 ** 40, page_size=2 ** 30) > 0
    assert all(n(B=b, table_width=w) % 8 == 0 for b in (1, 3) for w in (1, 7))
    p = decode(B=0, q=None, k_pages=None, v_pages=None, out=None, scratch=None)
    assert _lib.lib().vtx_paged_decode_attention(C.byref(p), None) == 0


def copy(src_pages, dst_pages, **kw):
    n = max(len(src_pages), 1)
    a, b, ptrs = (C.c_int64 * n)(*src_pages), (C.c_int64 * n)(*dst_pages), (C.c_void_p * 2)(16, 32)
    base = dict(pool_ptrs=C.cast(ptrs, C.c_void_p), src=C.cast(a, C.c_void_p), dst=C.cast(b, C.c_void_p), pools=2, pairs=len(src_pages), num_pages=10,
                page_bytes=64, page_stride_bytes=64)
    p = _lib.CopyPagesParams(**{**base, **kw})
    return _lib.lib().vtx_copy_pages(C.byref(p), None), _lib.last_error()


@pytest.mark.parametrize("src,dst,kw,text", [
    ([0], [10], {}, "pool of 10"), ([-1], [1], {}, "pool of 10"), ([0, 1], [5, 5], {}, "page 5 is written twice"),
    ([0, 1], [1, 2], {}, "both read and written"), ([3], [3], {}, "both read and written"), ([0], [1], dict(page_stride_bytes=63), "overlap"),
    ([0], [1], dict(pools=-1), "negative"), ([0], [1], dict(pool_ptrs=None), "null"), ([0], [1], dict(src=None), "null")])
def test_copy_pages_refusals(src, dst, kw, text):
    rc, msg = copy(src, dst, **kw)
    assert rc == -1 and text in msg


def test_copy_pages_of_nothing():
    assert copy([], [])[0] == 0 and copy([0], [1], pools=0)[0] == 0 and copy([0], [1], page_bytes=0, page_stride_bytes=0)[0] == 0
    assert _lib.lib().vtx_copy_pages(None, None) == -1


def test_cpu_tensors_are_rejected():
    x, pos = torch.zeros(2, 4, 64), torch.arange(2)
    fr, _ = attn_ops.rotary_inv_freq(64)
    table = torch.zeros(2, 1, dtype=torch.int32)
    pages = torch.zeros(2, 16, 4, 64)
    for f in (lambda: attn_ops.qk_norm_rotary(x, x, pos, fr), lambda: attn_ops.rotary_append(x, x, x, pos, pages, pages, table, fr),
              lambda: attn_ops.paged_decode_attention(x, pages, pages, table, table[:, 0]), lambda: attn_ops.copy_pages([pages], [0], [1])):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
    with pytest.raises(ValueError, match="2 sources for 1"):
        attn_ops.copy_pages([pages], [0, 1], [1])


def test_frequencies():
    f, s = attn_ops.rotary_inv_freq(8, 10000.0)
    assert f.dtype == torch.float64 and s == 1.0 and torch.allclose(f, torch.tensor([1, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    f2, _ = attn_ops.rotary_inv_freq(8, scaling="linear", factor=128)
    assert torch.equal(f2, f / 128)
    f3, _ = attn_ops.rotary_inv_freq(8, scaling="ntk", factor=16.0)
    assert f3[0] == 1 and abs(float(f3[-1] / f[-1]) - 1 / 16) < 1e-14
    f4, s4 = attn_ops.rotary_inv_freq(128, scaling="yarn", factor=8.0, trained_length=4096)
    f0, _ = attn_ops.rotary_inv_freq(128)
    turns = 4096 * f0 / (2 * math.pi)
    assert torch.equal(f4[turns > 32], f0[turns > 32]) and torch.equal(f4[turns < 1], f0[turns < 1] / 8)
    mid = (turns > 1) & (turns < 32)
    assert bool(((f4 < f0) & (f4 > f0 / 8))[mid].all()) and s4 == 0.1 * math.log(8) + 1
    assert attn_ops.rotary_inv_freq(2)[0].tolist() == [1.0]
    for kw in (dict(dim=7), dict(dim=0), dict(dim=8, factor=0), dict(dim=8, scaling="yarn"), dict(dim=2, scaling="ntk"),
               dict(dim=8, scaling="yarn", trained_length=64, slow=2, fast=1)):
        with pytest.raises(ValueError):
            attn_ops.rotary_inv_freq(**kw)
    with pytest.raises(NotImplementedError):
        attn_ops.rotary_inv_freq(8, scaling="other")


# ------------------------------------------------------------------ the cache's bookkeeping
@pytest.fixture
def host_copies(monkeypatch):
    """The pages copied as the kernel copies them, all at the same time, in tensors of the host."""
    from vortex_b200 import attn_ops

    def copy_pages(pools, src, dst):
        assert len(set(dst)) == len(dst) and not set(dst) & set(src)
        for p in pools:
            p[dst] = p[src]

    monkeypatch.setattr(attn_ops, "copy_pages", copy_pages)


def cache(**kw):
    from vortex_b200 import PagedKVCache
    base = dict(layers=2, num_pages=20, page_size=4, num_heads=1, head_dim=1, max_sequences=5, max_length=30, device="cpu", dtype=torch.float64)
    return PagedKVCache(**{**base, **kw})


def store(c, positions, rows, values):
    for p, r, x in zip(positions.tolist(), rows.tolist(), values):
        if p >= 0:
            at = c.block_table[r, p // c.page_size]
            for i, pool in enumerate(c.k + c.v):
                pool[at, p % c.page_size] = x + i


def held(c, row):
    n = c.length(row)
    at = torch.arange(n)
    return [pool[c.block_table[row].long()[at // c.page_size], at % c.page_size].flatten().tolist() for pool in c.k + c.v]


@pytest.mark.parametrize("seed", range(6))
def test_cache_holds_what_its_sequences_stored(host_copies, seed):
    """Random openings, growth, steps, forks, ends and compactions against lists of what each sequence stored."""
    import random
    rng = random.Random(seed)
    c, model, fresh = cache(page_size=rng.choice([1, 3, 4, 8])), {}, 0
    for _ in range(400):
        what = rng.choice(["open", "extend", "extend", "step", "step", "fork", "free", "compact"])
        rows = sorted(model)
        try:
            if what == "open":
                model[c.open()] = []
            elif what == "extend" and rows:
                some = rng.sample(rows, rng.randint(1, len(rows)))
                counts = [rng.randint(0, 6) for _ in some]
                pos, seq = c.extend(some, counts)
                vals = [1000.0 * (fresh + i) for i in range(sum(counts))]
                fresh += len(vals)
                store(c, pos, seq, vals)
                at = 0
                for r, n in zip(some, counts):
                    model[r] += vals[at:at + n]
                    at += n
            elif what == "step":
                some = None if rng.random() < 0.5 else rng.sample(rows, rng.randint(0, len(rows)))
                c.step(some)
                some = rows if some is None else some
                vals = [1000.0 * (fresh + i) for i in range(5)]
                fresh += 5
                store(c, c.positions, torch.arange(5), vals)
                for r in range(5):
                    if r in some:
                        model[r].append(vals[r])
                    assert c.lengths[r] == (len(model[r]) if r in some else 0)
                    assert c.positions[r] == (len(model[r]) - 1 if r in some else -1)
            elif what == "fork" and rows:
                r = rng.choice(rows)
                model[c.fork(r)] = list(model[r])
            elif what == "free" and rows:
                r = rng.choice(rows)
                c.free(r)
                del model[r]
            elif what == "compact":
                n = c.compact()
                assert n == 20 - c.unused_pages == len({p for r in model for p in c.pages(r)})
                assert all(p < n for r in model for p in c.pages(r))
        except (RuntimeError, ValueError) as e:
            assert "needed, " in str(e) or "rows hold" in str(e) or "tokens of at most" in str(e), e
        for r, vals in model.items():
            assert c.length(r) == len(vals) and held(c, r) == [[x + i for x in vals] for i in range(4)]
            assert c.block_table[r, len(c.pages(r)):].eq(-1).all()
        assert c.unused_pages + len({p for r in model for p in c.pages(r)}) == 20
    for r in list(model):
        c.free(r)
    assert c.unused_pages == 20 and c.block_table.eq(-1).all()


def test_cache_refusals_change_nothing(host_copies):
    c = cache(num_pages=3, max_sequences=2, max_length=9)
    a = c.open()
    c.extend([a], [6])
    before = (c.pages(a), c.length(a), c.unused_pages, c.block_table.clone())
    b = c.open()
    for f, exc in ((lambda: c.open(), RuntimeError), (lambda: c.extend([a], [4]), ValueError), (lambda: c.extend([a, a], [1, 1]), ValueError),
                   (lambda: c.extend([a, b], [1, 5]), RuntimeError), (lambda: c.extend([a], [-1]), ValueError), (lambda: c.extend([a], [1, 1]), ValueError),
                   (lambda: c.step([7]), ValueError), (lambda: c.fork(a), RuntimeError), (lambda: c.free(5), ValueError)):
        with pytest.raises(exc):
            f()
        assert (c.pages(a), c.length(a), c.unused_pages) == before[:3] and torch.equal(c.block_table, before[3]) and c.length(b) == 0
    c.free(b)
    with pytest.raises(ValueError, match="holds no sequence"):
        c.free(b)
    with pytest.raises(ValueError):
        cache(page_size=0)


@pytest.mark.parametrize("call", ["extend", "extend none", "step", "step some", "fork", "fork shared", "free", "compact"])
def test_cache_calls_that_fail_on_the_way_change_nothing(host_copies, monkeypatch, call):
    """Each upload and page copy of a call fails in turn: bookkeeping, table, positions and lengths are as before it, and the
    same call afterwards does what it would have done."""
    from vortex_b200 import attn_ops
    made = {"extend": lambda c: c.extend([0, 2], [6, 3]), "extend none": lambda c: c.extend([0], [0]), "step": lambda c: c.step(),
            "step some": lambda c: c.step([2]), "fork": lambda c: c.fork(0), "fork shared": lambda c: c.fork(2), "free": lambda c: c.free(0),
            "compact": lambda c: c.compact()}[call]

    def start():
        c = cache()
        for _ in range(3):
            c.open()
        pos, seq = c.extend([0, 1, 2], [7, 9, 8])
        store(c, pos, seq, [float(i) for i in range(24)])
        c.step([1])
        c.free(1)
        c.step([0])
        store(c, torch.tensor([7]), torch.tensor([0]), [30.0])
        return c

    def state(c):
        rows = [r for r, p in enumerate(c._pages) if p is not None]
        return (rows, [c.pages(r) for r in rows], [c.length(r) for r in rows], [held(c, r) for r in rows], sorted(c._unused), list(c._users),
                c.block_table.tolist(), c._table.tolist(), c.positions.tolist(), c.lengths.tolist())

    left = [None]

    def failing(f):
        def g(*a, **kw):
            if left[0] is not None:
                left[0] -= 1
                if left[0] < 0:
                    left[0] = None
                    raise RuntimeError("planted")
            return f(*a, **kw)
        return g

    for name in ("copy_", "to"):
        monkeypatch.setattr(torch.Tensor, name, failing(getattr(torch.Tensor, name)))
    monkeypatch.setattr(attn_ops, "copy_pages", failing(attn_ops.copy_pages))
    good = start()
    made(good)
    for n in range(10):
        c = start()
        before = state(c)
        left[0] = n
        try:
            made(c)
        except RuntimeError as e:
            assert str(e) == "planted"
            assert state(c) == before
            made(c)
            assert state(c) == state(good)
        else:
            left[0] = None
            break
    assert 0 < n < 10


def test_cache_step_without_a_sequence_that_ended(host_copies):
    """free between step and the decode step: the row is in the step no more, nor one that is opened in its place."""
    c = cache()
    a, b = c.open(), c.open()
    c.extend([a, b], [5, 3])
    c.step()
    assert c.positions.tolist() == [5, 3, -1, -1, -1] and c.lengths.tolist() == [6, 4, 0, 0, 0]
    c.free(a)
    assert c.positions.tolist() == [-1, 3, -1, -1, -1] and c.lengths.tolist() == [0, 4, 0, 0, 0]
    assert c.open() == a
    c.extend([a], [2])
    assert c.positions.tolist() == [-1, 3, -1, -1, -1] and c.lengths.tolist() == [0, 4, 0, 0, 0]
    c.step()
    assert c.positions.tolist() == [2, 4, -1, -1, -1] and c.lengths.tolist() == [3, 5, 0, 0, 0]


def test_cache_under_another_default_device(host_copies):
    """The host's side stays on the host."""
    with torch.device("meta"):
        c = cache()
        a = c.open()
        pos, seq = c.extend([a], [6])
        c.step()
        b = c.fork(a)
        c.free(a)
        assert c.compact() == 2
    assert all(t.device.type == "cpu" for t in (c._table, c.block_table, c.positions, pos, seq, *c.k))
    assert pos.tolist() == list(range(6)) and seq.tolist() == [a] * 6 and c.block_table[b, :2].tolist() == c.pages(b)
    assert c.positions[a] == -1 and c.length(b) == 7


def test_decode_attention_scratch_maximum():
    """More for a larger batch at one table width, and for other alignments; never beyond the header's maximum."""
    import itertools
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "include", "vortex_b200.h")) as f:
        n, shift = map(int, re.search(r"VTX_PAGED_DECODE_SCRATCH_MAX \((\d+) << (\d+)\)", f.read()).groups())
    f = _lib.lib().vtx_paged_decode_scratch_bytes
    need = lambda **kw: f(C.byref(decode(**kw)))  # noqa: E731
    assert need(B=1) < need(B=16) < need(B=256)
    assert need(B=64, q=16) != need(B=64, q=18)
    for io, D, (Hq, Hk), B, width, q, table in itertools.product((0, 1, 2), (1, 40, 64, 80, 128, 200, 256), ((1, 1), (8, 8), (12, 1), (16, 2), (600, 600)),
                                                                 (1, 7, 64, 5000), (1, 100, 1 << 20), (16, 18), (16, None)):
        assert 0 < need(io_dtype=io, D=D, Hq=Hq, Hk=Hk, B=B, table_width=width, q=q, block_table=table, num_pages=5000) <= n << shift


def test_a_sequence_read_back_in_order():
    """What a later chunk of a prompt attends to: a sequence's pages, flattened."""
    c = cache()
    a, b = c.open(), c.open()
    for n in (6, 5):
        pos, seq = c.extend([b, a], [n, n + 1])
        store(c, pos, seq, [100.0 * s + p for p, s in zip(pos.tolist(), seq.tolist())])
    assert c.k[0][c.pages(a)].flatten(0, 1)[:c.length(a)].flatten().tolist() == [100.0 * a + p for p in range(13)]
