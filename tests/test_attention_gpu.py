"""GPU: the attention-layer operators against their plain float64 forms (attn_ref.py), at the sizes, masks and layouts where
they can go wrong."""
import pytest
import torch

import attn_ref as R
from helpers import DT

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def A():
    from vortex_b200 import attn_ops, ops
    yield attn_ops
    ops.device_status()          # no test but those that say so leaves the status word set


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, ref, bound, label):
    assert got.shape == ref.shape
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), f"{label}: off by {float((err - bound).max()):.3e} beyond the bound, {float((err / bound).max()):.2f} times it"


def freqs(rot, base=10000.0):
    return (base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).cuda()


# heads, key heads, head size, rotated part: vectors (head and part in whole pairs of 16 bytes) and the general kernel
SHAPES = [(4, 2, 128, 128), (8, 1, 64, 32), (3, 3, 80, 80), (2, 2, 96, 64), (1, 1, 256, 256), (5, 2, 48, 16),
          (2, 1, 512, 512), (3, 2, 20, 6), (1, 2, 7, 2), (2, 1, 130, 130), (33, 2, 16, 16), (2, 2, 2, 2)]


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("Hq,Hk,D,rot", SHAPES)
@pytest.mark.parametrize("norm", ["none", "both", "q"])
def test_rotary(A, io, interleaved, Hq, Hk, D, rot, norm):
    g, dt = gen(1), DT[io]
    B, L = 2, 7
    qkv = torch.randn(B, L, Hq + Hk + 1, D, generator=g, device="cuda").to(dt)
    q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
    w = [None if norm == "none" or (norm == "q" and i) else (1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dt if i else torch.float32)
         for i in range(2)]
    pos = torch.tensor([[0, 1, 2, 1 << 20, 5, -3, 2 ** 31 - 1]] * B, device="cuda")[:, :L]
    pos[1] += torch.tensor([3, 0, 7, 1, 0, 0, -9], device="cuda")
    fr = freqs(rot)
    qo, ko = A.qk_norm_rotary(q, k, pos, fr, *w, eps=EPS, interleaved=interleaved, scale=1.25)
    for x, wi, y in ((q, w[0], qo), (k, w[1], ko)):
        ref, mag = R.norm_rotate(x.double(), wi, pos, fr, interleaved, 1.25, EPS)
        # (the reference's own angle, a product in float64, is off by |angle| 2^-53: 2.4e-7 rad at position 2^31)
        far = 4 * pos.abs().double()[..., None, None] * 2.0 ** -53
        within(y, ref, R.norm_rotate_bound(ref, mag, dt) + far * mag, "y")
        assert y.dtype == dt and y.is_contiguous()


def test_rotary_one_tensor_int32_positions_and_float32_frequencies(A):
    x = torch.randn(5, 3, 64, generator=gen(2), device="cuda")
    pos = torch.tensor([4, 0, 9, 2, 2], dtype=torch.int32, device="cuda")
    fr = freqs(64).float()
    y = A.qk_norm_rotary(x, None, pos, fr)
    ref, mag = R.norm_rotate(x.double(), None, pos, fr.double(), False, 1.0, 0)
    within(y, ref, R.norm_rotate_bound(ref, mag, torch.float32), "y")
    z = A.qk_norm_rotary(x.half(), None, pos, fr, interleaved=True)
    assert z.shape == x.shape and z.dtype == torch.float16


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("how", ["transposed", "expanded_positions", "odd_offset", "strided_head", "empty", "one_token"])
def test_rotary_layouts(A, io, how):
    g, dt, D = gen(3), DT[io], 64
    x = torch.randn(3, 4, 6, D, generator=g, device="cuda").to(dt)
    pos = torch.arange(4, device="cuda") + 11
    if how == "transposed":
        x = torch.randn(3, 6, 4, D, generator=g, device="cuda").to(dt).transpose(1, 2)
    elif how == "expanded_positions":
        pos = pos[None].expand(3, 4)
    elif how == "odd_offset":
        x = torch.randn(3 * 4 * 6 * D + 1, generator=g, device="cuda").to(dt)[1:].view(3, 4, 6, D)
    elif how == "strided_head":
        x = torch.randn(3, 4, 6, 2 * D, generator=g, device="cuda").to(dt)[..., ::2]
    elif how == "empty":
        x, pos = x[:, :0], pos[:0]
    elif how == "one_token":
        x, pos = x[:1, 3:], pos[3:]
    y = A.qk_norm_rotary(x, None, pos, freqs(D))
    ref, mag = R.norm_rotate(x.double(), None, pos.expand(x.shape[:2]), freqs(D), False, 1.0, 0)
    within(y, ref, R.norm_rotate_bound(ref, mag, dt), how)


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("H,D,rot", [(5, 64, 32), (33, 16, 16), (3, 20, 6), (2, 512, 512)])
def test_rotary_in_place_through_the_c_abi(A, io, H, D, rot):
    """The outputs are the inputs themselves: what the header allows and the wrapper does not use."""
    import ctypes as C

    from vortex_b200 import _lib
    g, dt = gen(25), DT[io]
    x, w = torch.randn(9, H, D, generator=g, device="cuda").to(dt), 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    pos, fr = torch.arange(9, device="cuda") * 777, freqs(rot)
    want = A.qk_norm_rotary(x, None, pos, fr, w, eps=EPS)
    at = dict(B=1, L=9, Hq=H, D=D, rot=rot, scale=1.0, eps=EPS, io_dtype={"f32": 0, "bf16": 1}[io], positions=pos.data_ptr(), positions_i64=1,
              pos_stride_l=1, inv_freq=fr.data_ptr(), inv_freq_f64=1, q_weight=w.data_ptr())
    for n in ("q", "q_out"):
        at.update({n: x.data_ptr(), n + "_stride_l": H * D, n + "_stride_h": D})
    _lib.check(_lib.lib().vtx_qk_norm_rotary_fwd(C.byref(_lib.RotaryParams(**at)), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert torch.equal(x, want)


def test_rotary_values_that_are_not_finite_stay_in_their_pair(A):
    x = torch.randn(1, 1, 64, generator=gen(4), device="cuda")
    x[0, 0, 3], x[0, 0, 40], x[0, 0, 63] = float("nan"), float("inf"), float("-inf")
    pos = torch.tensor([7], device="cuda")
    y = A.qk_norm_rotary(x, None, pos, freqs(32))          # pairs (i, i + 16), kept from 32 on
    hit = torch.zeros(64, dtype=torch.bool, device="cuda")
    hit[[3, 19, 40, 63]] = True
    assert bool((~y[0, 0].isfinite() == hit).all()) and torch.equal(y[0, 0, 40:], x[0, 0, 40:])
    w = torch.ones(64, device="cuda")                      # a norm reaches the whole head, and no other
    z = A.qk_norm_rotary(torch.cat([x, torch.ones_like(x)], 1), None, pos, freqs(32), w)
    assert bool(z[0, 0].isnan().any()) and bool(z[0, 1].isfinite().all())
    assert bool((A.qk_norm_rotary(torch.zeros_like(x), None, pos, freqs(32), w) == 0).all())


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("Hq,Hk,D,rot,L", [(4, 2, 128, 128, 9), (8, 1, 64, 32, 700), (5, 5, 80, 40, 33), (3, 2, 20, 6, 50), (2, 1, 256, 64, 3),
                                           (1, 1, 512, 512, 5), (33, 1, 16, 16, 130), (2, 2, 7, 2, 40), (2, 1, 130, 130, 3)])
@pytest.mark.parametrize("norm", ["none", "both", "k"])
def test_rotary_backward_against_the_formula(A, io, interleaved, Hq, Hk, D, rot, L, norm):
    g, dt = gen(5), DT[io]
    B = 2
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k = mk(B, L, Hq, D).to(dt).requires_grad_(), mk(B, L, Hk, D).to(dt).requires_grad_()
    wq = None if norm != "both" else (1 + 0.3 * mk(D)).to(dt).requires_grad_()
    wk = None if norm == "none" else (1 + 0.3 * mk(D)).requires_grad_()
    dq, dk = mk(B, Hq, L, D).to(dt).transpose(1, 2), mk(B, L, Hk, D).to(dt)
    pos = torch.randint(0, 100000, (B, L), generator=g, device="cuda", dtype=torch.int32)
    fr = freqs(rot)
    leaves = [t for t in (q, k, wq, wk) if t is not None]
    runs = []
    for _ in range(2):
        qo, ko = A.qk_norm_rotary(q, k, pos, fr, wq, wk, eps=EPS, interleaved=interleaved, scale=0.75)
        runs.append(torch.autograd.grad([qo, ko], leaves, [dq, dk]))
    assert all(torch.equal(a, b) for a, b in zip(*runs))    # sums in a fixed order
    grads = dict(zip([n for n, t in zip(("q", "k", "wq", "wk"), (q, k, wq, wk)) if t is not None], runs[0]))
    for n, x, w, dy in (("q", q, wq, dq), ("k", k, wk, dk)):
        dx, dw, mag, dwm = R.norm_rotate_bwd(dy.double(), x.detach().double(), None if w is None else w.detach(), pos, fr, interleaved, 0.75, EPS)
        # rotation and norm as in the forward, the norm's sums twice, the products of the second term (norm_rotate_bound: 26 u
        # for the one, 11 u for the other, 8 u)
        within(grads[n], dx, R.rounding(dx, dt) + 48 * R.U * mag, "d" + n)
        if w is not None:
            # a term as above (30 u), summed along a thread's rows, a block's rows, the blocks: fewer than rows + 64 additions
            rows = dwm.shape[0]
            within(grads["w" + n], dw, R.rounding(dw, w.dtype) + (30 + min(rows, 64) + rows / 64) * R.U * dwm.sum(0), "dw" + n)


def test_rotary_backward_against_differences(A):
    """Central differences of the operator itself, in fp32: f(x + h e) - f(x - h e) over 2 h, h = 2^-7, with f = sum(y dy)."""
    g = gen(6)
    L, H, D = 3, 2, 16
    q = torch.randn(L, H, D, generator=g, device="cuda")
    w = 1 + 0.3 * torch.randn(D, generator=g, device="cuda")
    dy = torch.randn(L, H, D, generator=g, device="cuda")
    pos, fr = torch.arange(L, device="cuda") * 1000, freqs(8)
    f = lambda q, w: float((A.qk_norm_rotary(q, None, pos, fr, w, eps=EPS).double() * dy.double()).sum())  # noqa: E731
    q1, w1 = q.clone().requires_grad_(), w.clone().requires_grad_()
    dq, dw = torch.autograd.grad(A.qk_norm_rotary(q1, None, pos, fr, w1, eps=EPS), [q1, w1], dy)
    h = 2.0 ** -7
    # the third derivative of x / |x|: a few / r^3 (r about 1, at least 0.5 for these rows) times |dy| sqrt(D) < 8, over 6 h^2;
    # fp32 values: 26 u sum |y dy| < 26 u 200 over h
    tol = 8 * 8 * 8 * h * h / 6 + 26 * R.U * 200 / h
    assert float(torch.sqrt((q * q).mean(-1)).min()) > 0.5
    for x, d, which in ((q, dq, 0), (w, dw, 1)):
        for i in range(0, x.numel(), 5):
            e = torch.zeros_like(x).view(-1)
            e[i] = h
            e = e.view_as(x)
            num = (f(q + e, w) - f(q - e, w)) / (2 * h) if which == 0 else (f(q, w + e) - f(q, w - e)) / (2 * h)
            assert abs(num - float(d.view(-1)[i])) <= tol


def test_rotary_one_gradient_wanted_and_unused_output(A):
    q = torch.randn(4, 2, 32, device="cuda", requires_grad=True)
    k = torch.randn(4, 1, 32, device="cuda")
    pos = torch.arange(4, device="cuda")
    qo, ko = A.qk_norm_rotary(q, k, pos, freqs(32))
    (dq,) = torch.autograd.grad(qo.sum(), q)
    back = A.qk_norm_rotary(torch.ones_like(q), None, -pos, freqs(32))
    assert torch.equal(dq, back)
    w = torch.ones(32, device="cuda", requires_grad=True)
    qo, ko = A.qk_norm_rotary(q.detach(), k, pos, freqs(32), None, w)
    (dw,) = torch.autograd.grad(qo.sum(), w)               # the queries do not pass through the keys' weight
    assert not bool(dw.any())
    with torch.no_grad():
        assert not A.qk_norm_rotary(q, k, pos, freqs(32))[0].requires_grad


def test_rotary_gradients_accumulate_into_leaves_and_through_a_graph(A):
    """backward() into .grad, twice through one graph, outputs changed in place, and gradients on a side stream."""
    g = gen(30)
    x = torch.randn(6, 3, 64, generator=g, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    pos, fr = torch.arange(6, device="cuda"), freqs(64)
    y = A.qk_norm_rotary(2 * x, None, pos, fr, w)
    z = (y * y).sum()
    z.backward(retain_graph=True)
    once = x.grad.clone(), w.grad.clone()
    z.backward()
    assert torch.equal(x.grad, 2 * once[0]) and torch.equal(w.grad, 2 * once[1])
    y = A.qk_norm_rotary(x, None, pos, fr, w)
    y.mul_(3.0)
    d1 = torch.autograd.grad(y.sum(), x)[0]
    d2 = torch.autograd.grad(A.qk_norm_rotary(x, None, pos, fr, w), x, torch.full_like(x, 3.0))[0]
    assert torch.equal(d1, d2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x2, w2 = x.detach().requires_grad_(), w.detach().requires_grad_()
        d3 = torch.autograd.grad(A.qk_norm_rotary(x2, None, pos, fr, w2), x2, torch.full_like(x, 3.0))[0]
    s.synchronize()
    assert torch.equal(d3, d2)
    y = A.qk_norm_rotary(x, None, pos, fr, w)
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_rotary_training_step_captured_into_a_graph(A):
    """Forward and backward through autograd inside a capture, replayed on other values."""
    g = gen(31)
    x = torch.randn(20, 4, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    pos, fr = torch.arange(20, device="cuda"), freqs(64)
    dy = torch.randn(20, 4, 64, generator=g, device="cuda").bfloat16()
    step = lambda: torch.autograd.grad(A.qk_norm_rotary(x, None, pos, fr, w), [x, w], dy)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step()
    with torch.no_grad():
        x.copy_(torch.randn(20, 4, 64, generator=g, device="cuda"))
    gr.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


# ------------------------------------------------------------------ cache
def pools(g, n, size, H, D, dt, layout="slots"):
    if layout == "heads":                      # [pages, heads, slots, D] seen as [pages, slots, heads, D]
        return [torch.randn(n, H, size, D, generator=g, device="cuda").to(dt).transpose(1, 2) for _ in range(2)]
    if layout == "joint":                      # keys and values side by side
        kv = torch.randn(n, size, 2, H, D, generator=g, device="cuda").to(dt)
        return [kv[:, :, 0], kv[:, :, 1]]
    if layout == "odd":                        # nothing on 16 bytes
        return [torch.randn(n * size * H * D + 1, generator=g, device="cuda").to(dt)[1:].view(n, size, H, D) for _ in range(2)]
    return [torch.randn(n, size, H, D, generator=g, device="cuda").to(dt) for _ in range(2)]


def make_table(g, lengths, size, extra=2):
    need = [-(-n // size) for n in lengths]
    order = torch.randperm(sum(need) + extra, generator=g, device="cuda").to(torch.int32)
    t = torch.full((len(lengths), max(need + [1]) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t, sum(need) + extra


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page,layout", [(16, "slots"), (1, "slots"), (5, "heads"), (64, "joint"), (16, "odd")])
@pytest.mark.parametrize("Hq,Hk,D,rot,norm", [(4, 2, 64, 64, False), (2, 2, 96, 32, True), (3, 1, 10, 4, True), (0, 2, 128, 0, False)])
def test_append(A, io, page, layout, Hq, Hk, D, rot, norm):
    g, dt = gen(7), DT[io]
    lengths = [1, 17, 0, 40]
    table, n = make_table(g, lengths, page)
    kp, vp = pools(g, n, page, Hk, D, dt, layout)
    k0, v0 = kp.clone(), vp.clone()
    # the last tokens of every sequence, without order, with two of padding between them
    rows = [(0, 0), (3, 39), (1, 16), (3, 38), (1, -1), (1, 15), (3, 0), (2, -5), (1, 3)]
    seq = torch.tensor([r for r, _ in rows], dtype=torch.int32, device="cuda")
    pos = torch.tensor([p for _, p in rows], device="cuda")
    T = len(rows)
    qkv = torch.randn(T, Hq + 2 * Hk, D, generator=g, device="cuda").to(dt)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]
    w = [(1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dt) if norm else None for _ in range(2)]
    fr = freqs(rot) if rot else None
    qo = A.rotary_append(q, k, v, pos, kp, vp, table, fr, *w, seq_ids=seq, eps=EPS)
    f64 = fr if rot else torch.zeros(0, dtype=torch.float64, device="cuda")
    ref, mag = R.norm_rotate(q.double(), w[0], pos, f64, False, 1.0, EPS)
    within(qo, ref, R.norm_rotate_bound(ref, mag, dt), "q")
    kref, kmag = R.norm_rotate(k.double(), w[1], pos, f64, False, 1.0, EPS)
    kb = R.norm_rotate_bound(kref, kmag, dt)
    for t, (s, p) in enumerate(rows):
        if p < 0:
            continue
        at = (int(table[s, p // page]), p % page)
        within(kp[at], kref[t], kb[t], "k")
        assert torch.equal(vp[at], v[t])
        k0[at], v0[at] = kp[at], vp[at]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)      # every other row as it was


def test_append_of_a_token_without_a_page(A):
    """Behind the table's width, in a row outside the table, at an entry outside the pool: stored nowhere, and reported."""
    from vortex_b200 import ops
    ops.device_status()
    table = torch.tensor([[0, -1], [7, 1]], dtype=torch.int32, device="cuda")
    fr = freqs(64)
    for rows in ([(0, 4)], [(0, 8)], [(1, 0)], [(2, 0)], [(-1, 0)], [(0, 2 ** 31 - 1)]):
        for D in (64, 7):
            kp, vp = (torch.zeros(3, 4, 2, D, device="cuda") for _ in range(2))
            x = torch.ones(2, 2, D, device="cuda")
            seq = torch.tensor([r for r, _ in rows] + [1], dtype=torch.int32, device="cuda")
            pos = torch.tensor([p for _, p in rows] + [5], device="cuda")
            A.rotary_append(x, x, x, pos, kp, vp, table, fr[:D // 2], seq_ids=seq)
            with pytest.raises(RuntimeError, match="block table"):
                ops.device_status()
            ops.device_status()
            vp[1, 1] = 0
            assert not bool(vp.any()) and int((kp != 0).any(-1).sum()) == 2


LENGTHS = [[1], [0, 3, 0], [16, 15, 17], [64, 63, 65, 1], [700], [0], [129, 2000, 5, 0, 333, 1]]


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("Hq,Hk,D", [(4, 4, 128), (8, 1, 64), (12, 1, 128), (20, 1, 64), (10, 2, 96), (6, 2, 256), (32, 1, 256), (2, 1, 40),
                                     (3, 3, 7), (2, 2, 80), (7, 1, 33), (16, 2, 200)])
@pytest.mark.parametrize("page,layout", [(16, "slots"), (48, "heads"), (1, "slots"), (5, "joint"), (256, "joint"), (16, "odd")])
def test_decode_attention(A, io, Hq, Hk, D, page, layout):
    dt = DT[io]
    for i, lengths in enumerate(LENGTHS):
        for window in (0, 1, 37):
            g = gen(100 + i)
            table, n = make_table(g, lengths, page)
            kp, vp = pools(g, n, page, Hk, D, dt, layout)
            q = 2 * torch.randn(len(lengths), Hq, D, generator=g, device="cuda").to(dt)
            lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
            out, lse = A.paged_decode_attention(q, kp, vp, table, lens, window=window, return_lse=True)
            ref, lref, bound = R.attend(q, kp, vp, table, lengths, D ** -0.5, window)
            within(out, ref, bound + R.rounding(ref.abs() + bound, dt), f"{lengths} window {window}")
            empty = lref == float("-inf")
            assert torch.equal(lse == float("-inf"), empty) and not bool(out[empty].any())
            # the sum's logarithm: a score's error, and its own rounding
            mag = (q.abs().amax() * kp.abs().amax()).double() * D ** 0.5
            assert float((lse - lref)[~empty].abs().max() if not bool(empty.all()) else 0) <= float((2 * D + 8) * R.U * mag + 2.0 ** -16)


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 20])
def test_decode_attention_contiguous_cache(A, io, D):
    """The reference's cache, [B, keys, 2, H, D] with keys and values side by side, of a length that is no multiple of 16."""
    g, dt, lengths = gen(8), DT[io], [50, 3, 0, 49]
    kv = torch.randn(4, 50, 2, 2, D, generator=g, device="cuda").to(dt)
    q = torch.randn(4, 6, 2 * D, generator=g, device="cuda").to(dt)[..., :D]
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = A.paged_decode_attention(q, kv[:, :, 0], kv[:, :, 1], None, lens, softmax_scale=0.2)
    ref, _, bound = R.attend(q, kv[:, :, 0], kv[:, :, 1], None, lengths, 0.2)
    within(out, ref, bound + R.rounding(ref.abs() + bound, dt), "out")


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("page", [16, 48, 3])
def test_decode_attention_reads_no_row_that_does_not_count(A, io, page):
    """NaN behind the last key, before the window, in pages of nobody: none reaches the output; table entries that no counted
    key needs may name no page."""
    g, dt, D = gen(9), DT[io], 128
    lengths, window = [100, 37, 1, 0], 30
    table, n = make_table(g, lengths, page)
    q = torch.randn(4, 4, D, generator=g, device="cuda").to(dt)
    good = pools(g, n, page, 2, D, dt)
    ref, _, bound = R.attend(q, *good, table, lengths, D ** -0.5, window)
    count = torch.zeros(n, page, dtype=torch.bool, device="cuda")
    bad_table = torch.full_like(table, 1 << 30)
    for b, m in enumerate(lengths):
        for j in range(max(0, m - window), m):
            count[int(table[b, j // page]), j % page] = True
            bad_table[b, j // page] = table[b, j // page]
    kp, vp = (torch.where(count[..., None, None], t, float("nan")) for t in good)
    out = A.paged_decode_attention(q, kp, vp, bad_table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), window=window)
    within(out, ref, bound + R.rounding(ref.abs() + bound, dt), "out")


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
def test_decode_attention_values_that_are_not_finite(A, io):
    """A value of infinity stays in its column, a key of infinity gives NaN as the formula does, elsewhere nothing changes."""
    g, dt, D, n = gen(10), DT[io], 64, 40
    q = torch.randn(2, 2, D, generator=g, device="cuda").to(dt)
    k, v = (torch.randn(2, n, 2, D, generator=g, device="cuda").to(dt) for _ in range(2))
    lens = torch.full((2,), n, dtype=torch.int32, device="cuda")
    clean = A.paged_decode_attention(q, k, v, None, lens)
    v[0, 5, 1, 9] = float("inf")
    q[1, 0, 3], k[1, 7, 0, 3] = 1.0, float("inf")
    out = A.paged_decode_attention(q, k, v, None, lens)
    assert float(out[0, 1, 9]) == float("inf") and bool(out[1, 0].isnan().all())
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[0, 1, 9] = False
    keep[1, 0] = False
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("Hq", [1, 16])
def test_decode_attention_many_light_keys_beside_a_heavy_one(A, io, Hq):
    """120,000 keys of 2^-25 of the heaviest one's weight together still weigh 2^-8 of it."""
    dt, D, n = DT[io], 64, 120000
    q = torch.zeros(1, Hq, D, device="cuda", dtype=dt)
    q[..., 0] = 1.0
    k = torch.zeros(1, n, 1, D, device="cuda", dtype=dt)
    v = torch.full_like(k, 64.0)
    for at in (0, n // 2, n - 1):
        kk, vv = k.clone(), v.clone()
        kk[0, at, 0, 0], vv[0, at] = 25.0, 0.0
        out = A.paged_decode_attention(q, kk, vv, None, torch.tensor([n], dtype=torch.int32, device="cuda"), softmax_scale=0.69314718055994531)
        w = (n - 1) * 2.0 ** -25
        ref = torch.full((1, Hq, D), 64.0 * w / (1 + w), dtype=torch.float64, device="cuda")
        # exact products and powers of two but for the scale's rounding (25 u of the exponent) and n / 64 sums a warp
        tol = R.rounding(ref, dt) + (2.0 ** -16 + (2 * 25 + n / 64 + 64) * 2 * R.U) * ref
        within(out, ref, tol, f"heavy key {at}")


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
def test_decode_attention_infinite_values_come_out_as_they_are(A, io):
    """At the heaviest key, whose probability is a power of two, at keys of any other weight, with either sign; both signs in a
    column, or a NaN, give NaN."""
    dt, D, n = DT[io], 64, 200
    g = gen(23)
    q, k, v = (torch.randn(1, m, h, D, generator=g, device="cuda").to(dt) for m, h in ((1, 2), (n, 1), (n, 1)))
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    top = torch.einsum("hd,nd->hn", q[0, 0].float(), k[0, :, 0].float()).argmax(-1)
    v[0, top[0], 0, 0] = float("inf")
    v[0, top[1], 0, 1] = float("-inf")
    for j in range(0, n, 3):
        v[0, j, 0, 2 + j % 20] = float("inf")
    v[0, 3, 0, 30], v[0, 4, 0, 30], v[0, 9, 0, 31] = float("inf"), float("-inf"), float("nan")
    out = A.paged_decode_attention(q[0], k, v, None, lens)
    ref, _, _ = R.attend(q[0], k, v, None, [n], D ** -0.5)
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(out.isposinf(), ref.isposinf()) and torch.equal(out.isneginf(), ref.isneginf())


def test_decode_attention_far_apart_scores(A):
    """Scores of +-1e4 and growing along the cache: the running maximum rises every few keys."""
    D, n = 64, 3000
    q = torch.ones(1, 8, D, device="cuda")
    k = (torch.arange(n, device="cuda")[None, :, None, None] - n / 2).expand(1, n, 1, D).contiguous() * 0.1
    v = torch.randn(1, n, 1, D, generator=gen(11), device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        for kk in (k, -k):
            a, b, c = q.to(dt), kk.to(dt), v.to(dt)
            out = A.paged_decode_attention(a, b, c, None, lens, softmax_scale=1.0)
            ref, _, bound = R.attend(a, b, c, None, [n], 1.0)
            within(out, ref, bound + R.rounding(ref.abs() + bound, dt), str(dt))


def test_decode_attention_keys_without_a_page(A):
    """An entry outside the pool, or a length behind the table's width: those keys are left out, and reported."""
    from vortex_b200 import ops
    ops.device_status()
    g = gen(12)
    for dt in (torch.bfloat16, torch.float32):
        for page in (16, 5):
            kp, vp = pools(g, 4, page, 1, 64, dt)
            q = torch.randn(2, 2, 64, generator=g, device="cuda").to(dt)
            good = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
            for entry in (-1, 4, 2 ** 31 - 1, -2 ** 31):
                t = good.clone()
                t[0, 0] = entry
                out = A.paged_decode_attention(q, kp, vp, t, torch.full((2,), 2 * page, dtype=torch.int32, device="cuda"))
                with pytest.raises(RuntimeError, match="block table"):
                    ops.device_status()
                part = A.paged_decode_attention(q, kp, vp, good, torch.full((2,), 2 * page, dtype=torch.int32, device="cuda"), window=page)
                # what is left: the second page's keys.  The sums differ in how they are dealt out
                ref, _, bound = R.attend(q, kp, vp, good, [2 * page] * 2, 0.125, page)
                within(out[:1], ref[:1], (bound + R.rounding(ref.abs() + bound, dt))[:1], "left")
                within(part[:1], ref[:1], (bound + R.rounding(ref.abs() + bound, dt))[:1], "window")
            out = A.paged_decode_attention(q, kp, vp, good, torch.tensor([2 * page, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
            with pytest.raises(RuntimeError, match="block table"):
                ops.device_status()
            ref, _, bound = R.attend(q, kp, vp, good, [2 * page] * 2, 0.125)
            within(out, ref, bound + R.rounding(ref.abs() + bound, dt), "width")
    neg = A.paged_decode_attention(q, kp, vp, good, torch.tensor([-5, -2 ** 31], dtype=torch.int32, device="cuda"))
    assert not bool(neg.any())
    ops.device_status()


@pytest.mark.parametrize("io,page", [("bf16", 16), ("f32", 3)])
def test_decode_attention_many_sequences(A, io, page):
    """More sequences than a block has threads, lengths from nothing on, and long ones among them."""
    g, dt, B = gen(13), DT[io], 300
    lengths = [(i * 37) % 61 if i % 100 else 900 for i in range(B)]
    table, n = make_table(g, lengths, page)
    kp, vp = pools(g, n, page, 2, 64, dt)
    q = torch.randn(B, 4, 64, generator=g, device="cuda").to(dt)
    out = A.paged_decode_attention(q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    ref, _, bound = R.attend(q, kp, vp, table, lengths, 0.125)
    within(out, ref, bound + R.rounding(ref.abs() + bound, dt), "out")


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hk,D", [(32, 32, 128), (600, 600, 64), (45, 15, 128), (14, 7, 80), (20, 20, 40), (74, 2, 64)])
def test_decode_attention_work_dealt_out(A, io, Hq, Hk, D):
    """Enough keys for every block of the machine: heads abreast or in a row, more heads than blocks, runs that end anywhere."""
    g, dt = gen(24), DT[io]
    for lengths in ([3000], [1500, 3, 0, 700], [257] * 9, [5000, 1, 1, 1]):
        table, n = make_table(g, lengths, 16)
        kp, vp = pools(g, n, 16, Hk, D, dt)
        q = torch.randn(len(lengths), Hq, D, generator=g, device="cuda").to(dt)
        out, lse = A.paged_decode_attention(q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), return_lse=True)
        ref, lref, bound = R.attend(q, kp, vp, table, lengths, D ** -0.5)
        within(out, ref, bound + R.rounding(ref.abs() + bound, dt), str(lengths))
        full = lref > float("-inf")
        # a score: (2 D + 8) u sum |q k| scale, at most 264 u 40 = 6e-4; the sum and its logarithm 1e-4
        assert torch.equal(lse > float("-inf"), full) and float((lse - lref)[full].abs().max()) < 1e-3


def test_decode_attention_offsets_beyond_32_bits(A):
    """A pool of more than 2^31 values (2^32 bytes): keys in its last pages."""
    D, page, n = 128, 256, (1 << 17) + 3
    kp, vp = (torch.zeros(n // 2, page, 1, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert kp.numel() > 1 << 31
    g = gen(14)
    last = torch.arange(n // 2 - 3, n // 2, dtype=torch.int32, device="cuda")
    kp[-3:], vp[-3:] = (torch.randn(3, page, 1, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = last[None]
    q = torch.randn(1, 4, D, generator=g, device="cuda").bfloat16()
    out = A.paged_decode_attention(q, kp, vp, table, torch.tensor([3 * page - 5], dtype=torch.int32, device="cuda"))
    ref, _, bound = R.attend(q, kp, vp, table, [3 * page - 5], D ** -0.5)
    within(out, ref, bound + R.rounding(ref.abs() + bound, torch.bfloat16), "out")
    k, v = (torch.randn(1, 1, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    A.rotary_append(q, k, v, torch.tensor([3 * page - 1], device="cuda"), kp, vp, table)
    assert torch.equal(kp[-1, -1], k[0]) and torch.equal(vp[-1, -1], v[0])


# ------------------------------------------------------------------ pages
@pytest.mark.parametrize("shape,dt", [((20, 16, 4, 32), torch.bfloat16), ((20, 3), torch.float32), ((20, 7), torch.bfloat16), ((20,), torch.uint8),
                                      ((20, 5, 8191), torch.float16), ((20, 0), torch.float32)])
@pytest.mark.parametrize("npools", [1, 3, 70])
def test_copy_pages(A, shape, dt, npools):
    g = gen(15)
    ps = [torch.randint(0, 255, shape, generator=g, device="cuda").to(dt) for _ in range(npools)]
    refs = [p.clone() for p in ps]
    src, dst = [3, 3, 0, 19, 7], [1, 2, 18, 5, 6]
    A.copy_pages(ps, src, torch.tensor(dst))
    for p, r in zip(ps, refs):
        r[dst] = r[src]
        assert torch.equal(p, r)
    A.copy_pages(ps, [], [])
    A.copy_pages([], [0], [1])


def test_copy_pages_many_pairs_pitched_and_offset(A):
    g = gen(16)
    base = torch.randint(0, 1 << 30, (5000, 40), generator=g, device="cuda")
    order = torch.randperm(5000, generator=g, device="cuda").cpu()
    for view in (lambda t: t[:, :32], lambda t: t[:, 1:], lambda t: t.int()[:, 1:36]):
        pool = view(base.clone())
        ref = pool.clone()
        src, dst = order[:2400], order[2400:4800]
        A.copy_pages([pool], src, dst)
        ref[dst.cuda()] = ref[src.cuda()]
        assert torch.equal(pool, ref)


# ------------------------------------------------------------------ streams, graphs, other callers
def test_operators_on_a_side_stream(A):
    g = gen(17)
    s = torch.cuda.Stream()
    kp, vp = pools(g, 8, 16, 2, 64, torch.bfloat16)
    kp0 = kp.clone()
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    qkv = torch.randn(2, 6, 64, generator=g, device="cuda").bfloat16()
    pos = torch.tensor([20, 63], device="cuda")
    lens = torch.tensor([21, 64], dtype=torch.int32, device="cuda")
    fr = freqs(64)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        A.copy_pages([kp, vp], [1], [7])
        q = A.rotary_append(qkv[:, :2], qkv[:, 2:4], qkv[:, 4:], pos, kp, vp, table, fr)
        out = A.paged_decode_attention(q, kp, vp, table, lens)
    assert torch.equal(kp, kp0) or s.query()            # nothing has run ahead of the stream
    s.synchronize()
    ref, _, bound = R.attend(q, kp, vp, table, [21, 64], 0.125)
    within(out, ref, bound + R.rounding(ref.abs() + bound, torch.bfloat16), "out")
    assert torch.equal(kp[7, :15], kp0[1, :15])


def test_captured_calls_follow_lengths_tables_and_positions(A):
    """Two graphs of the same step, replayed in turn on other lengths than they were captured with."""
    g = gen(18)
    kp, vp = pools(g, 40, 16, 2, 128, torch.bfloat16)
    table = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    pos = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    qkv = torch.randn(3, 8, 128, generator=g, device="cuda").bfloat16()
    fr = freqs(128)

    def step():
        q = A.rotary_append(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], pos, kp, vp, table, fr)
        return q, A.paged_decode_attention(q, kp, vp, table, lens)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = step()
        graphs.append((gr, res))
    order = torch.randperm(40, generator=g, device="cuda").to(torch.int32)
    table[:] = order[:36].view(3, 12)
    for i, lengths in enumerate(([1, 0, 190], [100, 17, 191], [180, 16, 192], [3, 150, 1])):
        lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        pos.copy_(lens - 1)
        qkv.normal_(generator=g)
        gr, (q, out) = graphs[i % 2]
        gr.replay()
        ref, _, bound = R.attend(q, kp, vp, table, lengths, 128 ** -0.5)
        within(out, ref, bound + R.rounding(ref.abs() + bound, torch.bfloat16), f"replay {i}")
        for b, n in enumerate(lengths):
            if n:
                assert torch.equal(vp[int(table[b, (n - 1) // 16]), (n - 1) % 16], qkv[b, 6:])


def test_two_decode_calls_at_once(A):
    """Calls on two streams share nothing: each has its own scratch."""
    g = gen(19)
    data = []
    for i in range(2):
        lengths = [3000 + 100 * i, 7, 1500]
        table, n = make_table(g, lengths, 16)
        kp, vp = pools(g, n, 16, 8, 128, torch.bfloat16)
        q = torch.randn(3, 8, 128, generator=g, device="cuda").bfloat16()
        data.append((q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), lengths))
    alone = [A.paged_decode_attention(*d[:5]) for d in data]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(A.paged_decode_attention(*data[i][:5]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])       # equal calls give equal bits


def test_backward_captured_into_a_graph(A):
    g = gen(20)
    q, k = torch.randn(40, 4, 64, generator=g, device="cuda").bfloat16(), torch.randn(40, 2, 64, generator=g, device="cuda").bfloat16()
    w = torch.ones(64, device="cuda")
    pos, fr = torch.arange(40, device="cuda"), freqs(64)
    from vortex_b200 import ops
    args = (q, k, pos, fr, w, w)
    want = ops.qk_norm_rotary_bwd(q, k, *args)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = ops.qk_norm_rotary_bwd(q, k, *args)
    gr.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


# ------------------------------------------------------------------ refusals of the wrappers
def test_refusals(A):
    x = torch.zeros(3, 4, 64, device="cuda")
    k = torch.zeros(3, 2, 64, device="cuda")
    pos, fr = torch.arange(3, device="cuda"), freqs(64)
    pages = torch.zeros(4, 16, 2, 64, device="cuda")
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    w = torch.ones(64, device="cuda")

    def refused(exc, text, f, *a, **kw):
        with pytest.raises(exc, match=text):
            f(*a, **kw)

    R_, P, D_ = A.qk_norm_rotary, A.rotary_append, A.paged_decode_attention
    refused(ValueError, "q must be", R_, x[0], None, pos, fr)
    refused(ValueError, "k must have", R_, x, k[:2], pos, fr)
    refused(ValueError, "k must have", R_, x, k.half(), pos, fr)
    refused(ValueError, "k must have", R_, x, k[..., :32], pos, fr)
    refused(ValueError, "positions have", R_, x, k, pos[:2], fr)
    refused(ValueError, "positions have", R_, x, k, pos[:, None], fr)
    refused(ValueError, "positions have", R_, x[None].expand(2, 3, 4, 64), None, pos[None].expand(3, 3), fr)
    refused(TypeError, "positions must", R_, x, k, pos.float(), fr)
    refused(TypeError, "inv_freq must", R_, x, k, pos, fr.half())
    refused(ValueError, "inv_freq must", R_, x, k, pos, freqs(66))
    refused(ValueError, "q_weight must", R_, x, k, pos, fr, w[:32])
    refused(ValueError, "k_weight without k", R_, x, None, pos, fr, None, w)
    refused(TypeError, "dtype", R_, x.double(), None, pos, fr)
    refused(RuntimeError, "CUDA", R_, x, k, pos.cpu(), fr)
    refused(NotImplementedError, "513", R_, torch.zeros(1, 1, 513, device="cuda"), None, pos[:1], fr)
    refused(ValueError, "v must have", P, x, k, k[:, :1], pos, pages, pages, table, fr)
    refused(ValueError, "k_pages must", P, x, k, k, pos, pages[:, :, :1], pages, table, fr)
    refused(ValueError, "v_pages must", P, x, k, k, pos, pages, pages.half(), table, fr)
    refused(ValueError, "unit stride", P, x, k, k, pos, pages.transpose(1, 3).contiguous().transpose(1, 3), pages, table, fr)
    refused(ValueError, "same pages", P, x, k, k, pos, pages, pages[:3], table, fr)
    refused(ValueError, "expanded", P, x, k, k, pos, pages[:, :1].expand(4, 16, 2, 64), pages, table, fr)
    refused(TypeError, "block_table must", P, x, k, k, pos, pages, pages, table.long(), fr)
    refused(ValueError, "block_table must", P, x, k, k, pos, pages, pages, table[0], fr)
    refused(ValueError, "one token for every row", P, x, k, k, pos, pages, pages, table[:2], fr)
    refused(ValueError, "seq_ids must", P, x, k, k, pos, pages, pages, table, fr, seq_ids=lens[:2])
    refused(TypeError, "seq_ids must", P, x, k, k, pos, pages, pages, table, fr, seq_ids=lens.long())
    refused(ValueError, "q must be", D_, x[0], pages, pages, table, lens)
    refused(ValueError, "k_pages must", D_, x, pages[0], pages, table, lens)
    refused(ValueError, "k_pages must", D_, x[..., :32], pages, pages, table, lens)
    refused(ValueError, "seqlens must", D_, x, pages, pages, table, lens[:2])
    refused(TypeError, "seqlens must", D_, x, pages, pages, table, lens.long())
    refused(ValueError, "block_table must", D_, x, pages, pages, table[:2], lens)
    refused(ValueError, "block_table must", D_, x, pages, pages, table[:, :0], lens)
    refused(ValueError, "without a block_table", D_, x, pages, pages, None, lens)
    refused(ValueError, "3 query heads for 2", D_, x[:, :3], pages, pages, table, lens)
    refused(ValueError, "window", D_, x, pages, pages, table, lens, window=-1)
    refused(NotImplementedError, "257", D_, torch.zeros(3, 2, 257, device="cuda"), *(torch.zeros(1, 4, 2, 257, device="cuda"),) * 2, table, lens)
    refused(ValueError, "one shape", A.copy_pages, [pages, pages[:2]], [0], [1])
    refused(ValueError, "contiguous", A.copy_pages, [pages[..., :32]], [0], [1])
    refused(ValueError, "written twice", A.copy_pages, [pages], [0, 1], [2, 2])
    refused(TypeError, "host data", A.copy_pages, [pages], pos[:1], [1])
    q = x.clone().requires_grad_()
    g1 = torch.autograd.grad(R_(q, None, pos, fr, w).sum(), q, create_graph=True)[0]
    refused(RuntimeError, "not have been used", lambda: torch.autograd.grad(g1.sum(), q, retain_graph=True))
    refused(RuntimeError, "differentiated once", lambda: g1.sum().backward())


# ------------------------------------------------------------------ a run of them together
@pytest.mark.parametrize("io,page", [("bf16", 16), ("f16", 5), ("f32", 16)])
@pytest.mark.parametrize("rotated,window", [(True, 0), (True, 20), (False, 0)])
def test_attention_layers_of_a_stack(A, io, page, rotated, window):
    """Two layers: ragged prompts, captured decode steps, a fork, a sequence that ends, a compaction and more steps; every
    output against softmax(q k) v in float64 over the keys and values as the layer stored them, which are checked apart."""
    from vortex_b200 import AttentionInferenceEngine, PagedKVCache

    g, dt, Hq, H, D, S = gen(21), DT[io], 6, 2, 64, 4
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    cache = PagedKVCache(2, 60, page, H, D, max_sequences=S, max_length=100, dtype=dt)
    fr, scale = A.rotary_inv_freq(32, 1e4, scaling="yarn", factor=4.0, trained_length=64)
    wq, wk = 1 + 0.2 * torch.randn(D, generator=g, device="cuda"), 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
    layers = [AttentionInferenceEngine(cache, i, fr if rotated else None, q_weight=wq if i else None, k_weight=wk if i else None, scale=scale,
                                       interleaved=bool(i), window=window) for i in range(2)]
    f64 = fr.cuda() if rotated else torch.zeros(0, dtype=torch.float64, device="cuda")
    seen = [{}, {}]                      # [layer][row] -> k (turned, float64, as stored) and v

    def turned(i, x, w, pos):
        y, mag = R.norm_rotate(x.double(), w if i else None, pos, f64, bool(i), scale, EPS)
        return y, R.norm_rotate_bound(y, mag, dt)

    def stored(i, row):
        n = cache.length(row)
        return R.gather(cache.k[i], cache.block_table[row], n), R.gather(cache.v[i], cache.block_table[row], n)

    def remember(i, row, k, pos, v):
        kk, vv = stored(i, row)
        y, b = turned(i, k, wk, pos)
        lo = cache.length(row) - k.shape[0]
        within(kk[lo:], y, b, "stored k")
        assert torch.equal(vv[lo:], v)
        if lo:
            assert torch.equal(kk[:lo], seen[i][row][0]) and torch.equal(vv[:lo], seen[i][row][1])
        seen[i][row] = (kk.clone(), vv.clone())

    rows, counts = [cache.open() for _ in range(3)], [33, 1, 16]
    pos, seq = cache.extend(rows, counts)
    for i, layer in enumerate(layers):
        q, k, v = mk(50, Hq, D), mk(50, H, D), mk(50, H, D)
        qo, ko = layer.prefill(q, k, v, pos, seq)
        y, b = turned(i, q, wq, pos)
        within(qo, y, b, "prompt q")
        at = 0
        for r, n in zip(rows, counts):
            assert torch.equal(ko[at:at + n], stored(i, r)[0])
            remember(i, r, k[at:at + n], pos[at:at + n], v[at:at + n])
            at += n

    q, k, v = ([torch.zeros(S, h, D, device="cuda", dtype=dt) for _ in range(2)] for h in (Hq, H, H))
    run = lambda: [layer.decode(q[i], k[i], v[i]) for i, layer in enumerate(layers)]  # noqa: E731
    cache.step([])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()

    def step(some=None):
        live = sorted(seen[0]) if some is None else some
        cache.step(some)
        for t in q + k + v:
            t.copy_(mk(*t.shape))
        graph.replay()
        lens = [cache.length(r) if r in live else 0 for r in range(S)]
        at = torch.tensor([max(n - 1, 0) for n in lens], device="cuda")
        for i in range(2):
            for r in live:
                remember(i, r, k[i][r:r + 1], at[r:r + 1], v[i][r:r + 1])
            y, b = turned(i, q[i], wq, at)
            ref, _, bound = R.attend(y, cache.k[i], cache.v[i], cache.block_table, lens, D ** -0.5, window)
            # the queries enter rounded: a change of q by b moves each score by at most sum b |k|, a probability by twice that
            for r in live:
                kk, vv = seen[i][r]
                lo = max(0, lens[r] - window) if window else 0
                kk, vv = kk[lo:].double().repeat_interleave(Hq // H, 1), vv[lo:].double().repeat_interleave(Hq // H, 1)
                d = torch.einsum("hd,nhd->hn", b[r], kk.abs()).amax(-1) * D ** -0.5
                bound[r] += 2 * torch.expm1(2 * d)[:, None] * vv.abs().amax(0)
            within(outs[i], ref, bound + R.rounding(ref.abs() + bound, dt), f"layer {i}")

    for _ in range(3):
        step()
    child = cache.fork(rows[0])
    for i in range(2):
        seen[i][child] = seen[i][rows[0]]
    step()
    step([rows[1], child])
    cache.free(rows[1])
    for i in range(2):
        del seen[i][rows[1]]
    assert cache.compact() == 60 - cache.unused_pages
    for i in range(2):
        for r in seen[i]:
            assert all(torch.equal(a, b) for a, b in zip(stored(i, r), seen[i][r]))
    for _ in range(2):
        step()


def test_cache_copies_on_the_current_stream(A):
    """fork and compact are work of the current stream: what was stored before them is in the copies."""
    from vortex_b200 import PagedKVCache
    s = torch.cuda.Stream()
    cache = PagedKVCache(1, 8, 4, 1, 8, max_sequences=3, max_length=16, dtype=torch.float32)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        a = cache.open()
        b = cache.open()
        pos, seq = cache.extend([a, b], [6, 2])
        x = torch.randn(8, 1, 8, generator=gen(22), device="cuda")
        torch.cuda._sleep(20_000_000)
        A.rotary_append(x, x, x, pos, cache.k[0], cache.v[0], cache.block_table, seq_ids=seq)
        c = cache.fork(a)
        cache.free(a)
        cache.compact()
        got = [R.gather(cache.k[0], cache.block_table[r], cache.length(r)) for r in (b, c)]
    s.synchronize()
    assert torch.equal(got[0], x[6:]) and torch.equal(got[1], x[:6])


@pytest.mark.parametrize("side", [0, 1])
def test_rotary_second_gradients_raise_on_every_path(A, side):
    """A gradient made with create_graph goes into what is differentiated again: an error wherever it depends on what is asked
    for, also where another path reaches that; what it does not depend on is not touched by it."""
    g = gen(40)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").requires_grad_()  # noqa: E731
    x, other, w, c = mk(5, 2, 64), mk(5, 2, 64), mk(64), mk(5, 2, 64)
    pos, fr = torch.arange(5, device="cuda"), freqs(64)
    qk = (lambda w: A.qk_norm_rotary(x, other, pos, fr, w)) if side == 0 else (lambda w: A.qk_norm_rotary(other, x, pos, fr, None, w))

    def once(f):
        with pytest.raises(RuntimeError, match="differentiated once"):
            f()

    y = qk(w)[side]
    plain = torch.autograd.grad(y, [x, w], c, retain_graph=True)
    gx, gw = torch.autograd.grad(y, [x, w], c, create_graph=True)
    assert torch.equal(gx, plain[0]) and torch.equal(gw, plain[1])
    for made in (gx, gw):
        loss = y.sum() + made.pow(2).sum() + other.sum()
        for leaf in (x, w, c):
            once(lambda: torch.autograd.grad(loss, leaf, retain_graph=True))
            once(lambda: torch.autograd.grad(made.sum(), leaf, retain_graph=True, allow_unused=True))
            once(lambda: loss.backward(inputs=[leaf], retain_graph=True))
        assert torch.equal(torch.autograd.grad(loss, other, retain_graph=True)[0], torch.ones_like(other))
    # the other tensor's gradient is no function of this one, its own values or their weight
    go = torch.autograd.grad(qk(w)[1 - side], other, c, create_graph=True)[0]
    assert torch.autograd.grad(go.sum(), [x, w], retain_graph=True, allow_unused=True) == (None, None)
    once(lambda: torch.autograd.grad(go.sum(), c, retain_graph=True))
    # a rotation alone is linear: its gradient depends on the output's, not on the values
    y = qk(None)[side]
    gx = torch.autograd.grad(y, x, c, create_graph=True)[0]
    once(lambda: torch.autograd.grad(gx.sum(), c, retain_graph=True))
    assert torch.equal(torch.autograd.grad(y.sum() + gx.pow(2).sum(), x, retain_graph=True)[0], torch.autograd.grad(qk(None)[side].sum(), x)[0])
    gx = torch.autograd.grad(y.pow(2).sum(), x, create_graph=True)[0]          # (here the output's gradient is one of the values)
    once(lambda: torch.autograd.grad(y.sum() + gx.pow(2).sum(), x))
    y = qk(w)[side]
    gx = torch.autograd.grad(y.sum(), x, create_graph=True)[0]
    once(lambda: (y.sum() + gx.pow(2).sum()).backward())
    assert not torch.autograd.grad(qk(w)[side].sum(), x)[0].requires_grad


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("D", [64, 128, 40])
def test_decode_attention_of_no_key_at_all(A, io, page, D):
    """A sequence whose counted keys all lie in pages that the table does not give: zeros and -inf, as for one of length 0,
    finished by one block (short) or joined from several (long).  Keys that are there and whose scores are all -inf: the formula's
    0 / 0.  Some of each: the others' softmax."""
    from vortex_b200 import ops
    ops.device_status()
    g, dt, H = gen(43), DT[io], 2
    kp, vp = pools(g, 300, page, 1, D, dt)
    width = 1200 // page
    order = torch.randperm(300, generator=g, device="cuda").to(torch.int32)
    q = torch.randn(4, H, D, generator=g, device="cuda").to(dt)
    for n, window in ((3, 0), (1200 // page * page, 0), (1000, 900)):
        table = torch.stack([order[:width], torch.full((width,), -1, device="cuda", dtype=torch.int32), order[-width:].flip(0),
                             torch.full((width,), 300, device="cuda", dtype=torch.int32)])
        if window:
            table[1, :(n - window) // page] = 7                  # pages before the window are there and do not count
        lens = torch.tensor([n, n, 0, n], dtype=torch.int32, device="cuda")
        out, lse = A.paged_decode_attention(q, kp, vp, table, lens, window=window, return_lse=True)
        with pytest.raises(RuntimeError, match="block table"):
            ops.device_status()
        ref, _, bound = R.attend(q[:1], kp, vp, table[:1], [n], D ** -0.5, window)
        within(out[:1], ref, bound + R.rounding(ref.abs() + bound, dt), "first")
        assert not bool(out[1:].any()) and bool(lse[1:].isneginf().all()) and bool(lse[0].isfinite().all())
    # scores of -inf: a key of -inf in a value where every query is 1, the others 0
    q[..., 0] = 1.0
    table[1], table[2], table[3] = order[:width], order[:width], order[:width]
    for n in (3, 1200 // page * page):
        kk = kp.clone()
        kk[..., 0] = float("-inf")
        lens = torch.tensor([n, n, n, n], dtype=torch.int32, device="cuda")
        table[3] = -1
        table[3, 0] = order[0]
        out, lse = A.paged_decode_attention(q, kk, vp, table, lens, return_lse=True)
        if n > page:
            with pytest.raises(RuntimeError, match="block table"):
                ops.device_status()
        assert bool(out.isnan().all()) and bool(lse.isneginf().all())
        kk = kp.clone()
        kk[order[0].long(), 0, :, 0] = float("-inf")            # one key, the first of each, beside finite ones
        out, lse = A.paged_decode_attention(q[:1], kk, vp, table[:1], lens[:1], return_lse=True)
        ref, _, bound = R.attend(q[:1], kp, vp, table[:1], [n], D ** -0.5, n - 1)
        within(out, ref, bound + R.rounding(ref.abs() + bound, dt), "rest")
        assert bool(lse.isfinite().all())
    ops.device_status()


def test_rotary_refuses_forward_mode_derivatives(A):
    """A tangent would be lost: the call says so, with and without gradients recorded; duals nearby do not matter."""
    import torch.autograd.forward_ad as fwd
    g = gen(41)
    x, w = torch.randn(3, 2, 64, generator=g, device="cuda"), torch.ones(64, device="cuda")
    pos, fr = torch.arange(3, device="cuda"), freqs(64)
    want = A.qk_norm_rotary(x, x, pos, fr, w, w)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        dx, dw, df = dual(x), dual(w), dual(fr)
        for args in ((dx, x, pos, fr, w, w), (x, dx, pos, fr, w, w), (x, x, pos, fr, dw, w), (x, x, pos, fr, w, dw), (x, x, pos, df),
                     (dx, None, pos, fr)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                A.qk_norm_rotary(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                A.qk_norm_rotary(*args)
        got = A.qk_norm_rotary(x, x, pos, fr, w, w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_written_pools_say_so_to_autograd(A):
    """A call that writes pools raises their version (views of one tensor share it): a product that saved one before and is
    differentiated after raises instead of using what lies there by then.  Pools made in inference mode have no version."""
    g = gen(42)
    kv = torch.randn(4, 16, 2, 2, 64, generator=g, device="cuda")
    kp, vp = kv[:, :, 0], kv[:, :, 1]
    x = torch.randn(2, 2, 64, generator=g, device="cuda")
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    calls = {"append": lambda k, v: A.rotary_append(x, x, x, pos, k, v, table), "copy": lambda k, v: A.copy_pages([k, v], [0], [2])}
    a = torch.ones(4, 16, 2, 64, device="cuda", requires_grad=True)
    for name, call in calls.items():
        for k, v in ((kp, vp), (torch.zeros(4, 16, 2, 64, device="cuda"), torch.zeros(4, 16, 2, 64, device="cuda"))):
            if name == "copy":
                k, v = k.contiguous().clone(), v.contiguous().clone()
            before, saved = (k._version, v._version), ((a * k).sum(), (a * v).sum())
            call(k, v)
            assert k._version > before[0] and v._version > before[1], name
            for s in saved:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    s.backward()
        with torch.inference_mode():
            k, v = (torch.zeros(4, 16, 2, 64, device="cuda") for _ in range(2))
            call(k, v)
        call(k, v)
    q = torch.randn(2, 2, 64, generator=g, device="cuda")
    lens = torch.tensor([4, 5], dtype=torch.int32, device="cuda")
    kp, vp = kp.contiguous(), vp.contiguous()
    before = kp._version, vp._version, q._version
    A.paged_decode_attention(q, kp, vp, table, lens)
    A.qk_norm_rotary(q, None, pos, freqs(64))
    assert (kp._version, vp._version, q._version) == before


def test_cache_refuses_to_change_under_capture(A):
    """Its uploads would not be part of the graph: refused before anything is changed, the capture goes on and replays."""
    from vortex_b200 import AttentionInferenceEngine, PagedKVCache
    cache = PagedKVCache(1, 8, 4, 1, 64, max_sequences=3, max_length=16)
    layer = AttentionInferenceEngine(cache, 0, A.rotary_inv_freq(64)[0])
    a, b = cache.open(), cache.open()
    cache.extend([a, b], [4, 3])
    cache.step([a])
    x = torch.randn(3, 1, 64, generator=gen(44), device="cuda").bfloat16()
    eager = layer.decode(x, x, x)
    torch.cuda.synchronize()
    now = lambda: ([cache.pages(r) for r in (a, b)], [cache.length(r) for r in (a, b)], cache.unused_pages)  # noqa: E731
    before, device = now(), (cache.block_table.clone(), cache.positions.clone(), cache.lengths.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for f in (cache.step, lambda: cache.step([b]), lambda: cache.extend([a], [2]), lambda: cache.fork(b), lambda: cache.free(a), cache.compact):
            with pytest.raises(RuntimeError, match="capture"):
                f()
            assert now() == before
        out = layer.decode(x, x, x)
    assert now() == before and all(torch.equal(p, q) for p, q in zip(device, (cache.block_table, cache.positions, cache.lengths)))
    graph.replay()
    assert torch.equal(out, eager)


def test_a_sequence_that_ends_between_step_and_decode(A):
    """Its row stores nothing, gives zeros and reports nothing; the others are as without it."""
    from vortex_b200 import AttentionInferenceEngine, PagedKVCache, ops
    ops.device_status()
    g = gen(45)
    cache = PagedKVCache(1, 8, 4, 1, 64, max_sequences=3, max_length=16)
    layer = AttentionInferenceEngine(cache, 0, A.rotary_inv_freq(64)[0])
    a, b = cache.open(), cache.open()
    pos, seq = cache.extend([a, b], [6, 5])
    x, y = (torch.randn(n, 1, 64, generator=g, device="cuda").bfloat16() for n in (11, 3))
    layer.prefill(x, x, x, pos, seq)
    cache.step()
    want = layer.decode(y, y, y)
    cache.free(a)
    got = layer.decode(y, y, y)                 # the same step again, without the first row
    ops.device_status()
    assert not bool(got[a].any()) and torch.equal(got[b], want[b])
