"""The operators of a striped stack's attention layers, as cases that can be timed and compared.

A striped stack keeps an attention layer after every few Hyena layers (five of the 32 layers of the 7B-shaped stack of
``bench.py``: hidden size 4096, 32 heads of 128; hidden size 8192 for the 40B-shaped one, whose 64 heads are 8 per GPU on
8 GPUs).  Four operators serve and train them beside the projections:

* ``rotary``: positions by rotation, optionally behind an RMS norm of each head, forward and backward;
* ``append``: the same on the queries and keys of new tokens, keys and values stored in the pages of a cache;
* ``attend``: one new token of every sequence against the pages of that cache;
* ``pages``: pages copied inside a cache, where a sequence is forked or the cache is compacted.

``run`` computes them with elementary torch operations in fp32 (angles in fp64) or, with ``own`` set, through
``vortex_b200.attn_ops``; ``exact`` evaluates the definitions in fp64.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
MOST_KEYS = 1 << 20             # keys x key heads / 8 of the largest cache that is read
HEADS = ((32, 32), (32, 8), (16, 16), (16, 2), (8, 8), (8, 1), (64, 8), (5, 5), (12, 4))


def listed():
    return [
        # one decode step of 64 sequences, far into long contexts (positions interpolated by a factor of 128)
        dict(name="rotary_decode_b64", op="rotary", B=64, L=1, Hq=32, Hk=32, D=128, rot=128, interleaved=False, norm=False,
             train=False, dtype="bf16", far=1 << 20, factor=128.0),
        # queries and keys of a batch prefill of 4 x 8192 tokens (the batch of bench.py's default workload)
        dict(name="rotary_prefill", op="rotary", B=4, L=8192, Hq=32, Hk=32, D=128, rot=128, interleaved=False, norm=False,
             train=False, dtype="bf16", far=0, factor=1.0),
        # a training step with normed heads and shared key heads: forward, and all four gradients
        dict(name="norm_rotary_train", op="rotary", B=2, L=8192, Hq=32, Hk=8, D=128, rot=128, interleaved=True, norm=True,
             train=True, dtype="bf16", far=0, factor=1.0),
        # the same in fp32 at an odd length, few heads, a part of each head rotated
        dict(name="norm_rotary_train_odd", op="rotary", B=1, L=1003, Hq=5, Hk=5, D=80, rot=40, interleaved=False, norm=True,
             train=True, dtype="f32", far=0, factor=1.0),
        # one decode step of 64 sequences: the new keys and values go to the last page of each
        dict(name="append_decode_b64", op="append", B=64, longest=512, new=1, Hq=32, Hk=32, D=128, rot=128, interleaved=False,
             norm=False, dtype="bf16", page=16),
        # ragged prompts stored behind what their sequences hold already, normed heads, shared key heads
        dict(name="append_prompts", op="append", B=13, longest=4096, new=1500, Hq=32, Hk=8, D=128, rot=64, interleaved=True,
             norm=True, dtype="bf16", page=64),
        # the interactive decode step: one short sequence
        dict(name="attend_b1", op="attend", B=1, shortest=700, longest=700, Hq=32, Hk=32, D=128, dtype="bf16", page=16, window=0),
        # the serving decode step: 64 sequences behind a prompt of 8192 tokens, a key head for every query head
        dict(name="attend_b64", op="attend", B=64, shortest=8192, longest=8704, Hq=32, Hk=32, D=128, dtype="bf16", page=16, window=0),
        # one GPU's heads of a sequence of 1,048,576 tokens: few rows, one long axis
        dict(name="attend_1m", op="attend", B=1, shortest=1048576, longest=1048576, Hq=8, Hk=8, D=128, dtype="bf16", page=256, window=0),
        # continuous batching: lengths from nothing to long, shared key heads, smaller heads, a sliding window
        dict(name="attend_ragged", op="attend", B=48, shortest=0, longest=32768, Hq=32, Hk=8, D=64, dtype="f16", page=48, window=20000),
        # one sequence forked: its last page copied in K and V of the five attention layers
        dict(name="pages_fork", op="pages", pages=64, copies=1, pools=10, page_bytes=131072),
        # a cache compacted after sequences ended
        dict(name="pages_compact", op="pages", pages=2048, copies=701, pools=10, page_bytes=131072),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "pages"])
    if op == "pages":
        page_bytes = rng.choice([4096, 16384, 65536, 131072, 262144])
        pools = rng.randint(2, 10)
        pages = _log(rng, 16, 268435456 // page_bytes)
        return dict(op=op, pages=pages, copies=_log(rng, 1, max(1, pages // 3)), pools=pools, page_bytes=page_bytes)
    Hq, Hk = rng.choice(HEADS)
    D = rng.choice([64, 80, 96, 128, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    case = dict(op=op, Hq=Hq, Hk=Hk, D=D, dtype=dtype)
    if op == "attend":
        page = rng.choice([1, 16, 16, 48, 64, 256])
        keys = MOST_KEYS * 8 // Hk * 128 // D // (2 if dtype == "f32" else 1)
        longest = _log(rng, 1, min(keys, 1 << 20))
        B = _log(rng, 1, max(1, min(256, keys // longest)))
        shortest = rng.choice([0, longest // 2, longest])
        if page == 1 and longest * B > 1 << 18:
            page = 16
        return dict(case, B=B, shortest=shortest, longest=longest, page=page,
                    window=rng.choice([0, 0, 0, max(1, longest // 3)]))
    case.update(rot=rng.choice([D, D, D // 2 // 2 * 2]), interleaved=rng.random() < 0.5, norm=rng.random() < 0.5)
    top = 32768 * 64 * 128 * 2 // ((Hq + Hk) * D * BYTES[dtype])
    if op == "rotary":
        case["train"] = rng.random() < 0.5
        L = _log(rng, 1, top // (5 if case["train"] else 1))
        B = _log(rng, 1, max(1, min(64, top // (5 if case["train"] else 1) // L)))
        return dict(case, B=B, L=L, far=rng.choice([0, 0, 1 << 20]), factor=rng.choice([1.0, 4.0, 128.0]))
    new = rng.choice([1, 1, _log(rng, 2, 2048)])
    B = _log(rng, 1, max(1, min(128, top // 4 // new)))
    longest = new + _log(rng, 1, max(2, min(8192, 65536 // B)))
    return dict(case, B=B, longest=longest, new=new, page=rng.choice([1, 16, 48, 64, 256]) if longest * B < 1 << 16 else 16)


def _spread(n, lo, hi):
    """n whole numbers spread evenly from hi down to lo, both included."""
    return [hi - i * (hi - lo) // max(1, n - 1) for i in range(n)]


def _lengths(g, n, lo, hi):
    """The same without order (another seed: another order); a list, as the host keeps it."""
    values = _spread(n, lo, hi)
    return [values[i] for i in torch.randperm(n, generator=g).tolist()]


def _inv_freq(rot, factor):
    return (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot) / factor).cuda()


def _tables(g, lengths, page):
    """Pages of each sequence, drawn without order from a pool a little larger than they need; unused entries are -1."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, dtype=torch.int64).to(torch.int32)
    table = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table.cuda(), total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)

    def randn(*shape, dtype):
        return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)

    s = {"case": case}
    if case["op"] == "pages":
        n, words = case["pages"], case["page_bytes"] // 2
        s["pools"] = [randn(n, words, dtype=torch.bfloat16) for _ in range(case["pools"])]
        order = torch.randperm(n, generator=host).tolist()
        c = case["copies"]
        s["src"], s["dst"] = order[:c], order[c:2 * c]
        return s
    dt, Hq, Hk, D = DT[case["dtype"]], case["Hq"], case["Hk"], case["D"]
    if case["op"] == "attend":
        lengths = _lengths(host, case["B"], case["shortest"], case["longest"])
        s["table"], total = _tables(host, lengths, case["page"])
        s["lengths"] = lengths
        s["seqlens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q"] = 2 * randn(case["B"], Hq, D, dtype=dt)
        s["k_pages"], s["v_pages"] = (randn(total, case["page"], Hk, D, dtype=dt) for _ in range(2))
        return s
    s["inv_freq"] = _inv_freq(case["rot"], case.get("factor", 1.0))
    s["wq"] = s["wk"] = None
    if case["norm"]:
        s["wq"], s["wk"] = ((1 + 0.2 * randn(D, dtype=torch.float32)).to(dt) for _ in range(2))
    if case["op"] == "rotary":
        B, L = case["B"], case["L"]
        # slices of the packed projection output, as a model has them
        qkv = randn(B, L, Hq + 2 * Hk, D, dtype=dt)
        s["q"], s["k"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
        first = torch.tensor(_lengths(host, B, 0, case["far"]), device="cuda")[:, None]
        s["positions"] = (first + torch.arange(L, device="cuda")).to(torch.int32)
        if case["train"]:
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
            if case["norm"]:
                s["wq"].requires_grad_(), s["wk"].requires_grad_()
            s["dq"], s["dk"] = randn(B, L, Hq, D, dtype=dt), randn(B, L, Hk, D, dtype=dt)
        return s
    lengths = _lengths(host, case["B"], case["new"], case["longest"])
    s["table"], total = _tables(host, lengths, case["page"])
    fresh = [case["new"]] * case["B"]
    if case["new"] > 1:                                          # ragged prompts, each at least one token
        fresh = _lengths(host, case["B"], 1, case["new"])
    s["positions"] = torch.cat([torch.arange(m - n, m) for n, m in zip(fresh, lengths)]).to(torch.int32).cuda()
    s["seq_ids"] = torch.repeat_interleave(torch.arange(case["B"]), torch.tensor(fresh)).to(torch.int32).cuda()
    T = sum(fresh)
    qkv = randn(T, Hq + 2 * Hk, D, dtype=dt)
    s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]
    s["k_pages"], s["v_pages"] = (randn(total, case["page"], Hk, D, dtype=dt) for _ in range(2))
    return s


def _norm_rotate(x, w, positions, inv_freq, interleaved):
    """x [..., heads, D] in fp32: normed by its root mean square and the weight (where there is one), then rotated."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    angle = positions.double()[..., None, None] * inv_freq
    c, sn = angle.cos().float(), angle.sin().float()
    rot = 2 * inv_freq.numel()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * c - b * sn, a * sn + b * c], -1)
    return y if rot == x.shape[-1] else torch.cat([y, x[..., rot:]], -1)


def _plain_attend(s):
    c = s["case"]
    out = torch.zeros_like(s["q"])
    step = max(1, (1 << 28) // (c["Hk"] * c["D"]))          # keys taken to fp32 at a time: 1 GiB of each
    for b, n in enumerate(s["lengths"]):
        first = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            continue
        q = s["q"][b].float().view(c["Hk"], -1, c["D"]) * c["D"] ** -0.5
        top, total, acc = None, 0.0, 0.0
        for lo in range(first, n, step):
            at = torch.arange(lo, min(n, lo + step), device="cuda")
            page, slot = s["table"][b].long()[at // c["page"]], at % c["page"]
            k = s["k_pages"][page, slot].float()
            score = q @ k.permute(1, 2, 0)
            del k
            best = score.amax(-1, keepdim=True)
            new = best if top is None else torch.maximum(top, best)
            p = (score - new).exp()
            keep = 0.0 if top is None else (top - new).exp()
            v = s["v_pages"][page, slot].float()
            acc = acc * keep + p @ v.permute(1, 0, 2)
            total = total * keep + p.sum(-1, keepdim=True)
            top = new
        out[b] = (acc / total).reshape(c["Hq"], c["D"]).to(out.dtype)
    return out


def run(s):
    c = s["case"]
    if own:
        return _run_own(s)
    if c["op"] == "pages":
        src, dst = torch.tensor(s["src"], device="cuda"), torch.tensor(s["dst"], device="cuda")
        for pool in s["pools"]:
            pool[dst] = pool[src]
        return s["pools"]
    if c["op"] == "attend":
        return _plain_attend(s)
    dt = DT[c["dtype"]]
    qo, ko = (_norm_rotate(s[x].float(), s["w" + x], s["positions"], s["inv_freq"], c["interleaved"]).to(dt) for x in "qk")
    if c["op"] == "append":
        at = s["positions"].long()
        page, slot = s["table"].long()[s["seq_ids"].long(), at // c["page"]], at % c["page"]
        s["k_pages"][page, slot] = ko
        s["v_pages"][page, slot] = s["v"]
        return qo, s["k_pages"], s["v_pages"]
    if not c["train"]:
        return qo, ko
    leaves = [s["q"], s["k"]] + ([s["wq"], s["wk"]] if c["norm"] else [])
    return (qo.detach(), ko.detach(), *torch.autograd.grad([qo, ko], leaves, [s["dq"], s["dk"]]))


def _run_own(s):
    from vortex_b200 import attn_ops

    c = s["case"]
    if c["op"] == "pages":
        attn_ops.copy_pages(s["pools"], s["src"], s["dst"])
        return s["pools"]
    if c["op"] == "attend":
        return attn_ops.paged_decode_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["seqlens"], window=c["window"])
    if c["op"] == "append":
        q = attn_ops.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["k_pages"], s["v_pages"], s["table"],
                                   s["inv_freq"], s["wq"], s["wk"], seq_ids=None if c["new"] == 1 else s["seq_ids"],
                                   eps=EPS, interleaved=c["interleaved"])
        return q, s["k_pages"], s["v_pages"]
    q, k = attn_ops.qk_norm_rotary(s["q"], s["k"], s["positions"], s["inv_freq"], s["wq"], s["wk"], eps=EPS,
                                   interleaved=c["interleaved"])
    if not c["train"]:
        return q, k
    leaves = [s["q"], s["k"]] + ([s["wq"], s["wk"]] if c["norm"] else [])
    return (q.detach(), k.detach(), *torch.autograd.grad([q, k], leaves, [s["dq"], s["dk"]]))


def work(case):
    if case["op"] == "pages":
        return {"bytes": 2 * case["copies"] * case["pools"] * case["page_bytes"], "flops": 0}
    e, Hq, Hk, D = BYTES[case["dtype"]], case["Hq"], case["Hk"], case["D"]
    if case["op"] == "attend":
        lengths = _spread(case["B"], case["shortest"], case["longest"])
        keys = sum(min(n, case["window"]) if case["window"] else n for n in lengths)
        return {"bytes": 2 * keys * Hk * D * e + 2 * case["B"] * Hq * D * e, "flops": 4 * keys * Hq * D}
    ops = 4 * case["rot"] // 2 + (4 * D if case["norm"] else 0)       # rotation: 4 products and 2 sums a pair; norm: 4 a value
    if case["op"] == "rotary":
        rows = case["B"] * case["L"] * (Hq + Hk)
        if not case["train"]:
            return {"bytes": 2 * rows * D * e, "flops": rows * ops}
        # forward: x in, y out; backward: dy in, dx out, and x again where the norm's gradient needs it
        return {"bytes": (5 if case["norm"] else 4) * rows * D * e, "flops": rows * ops * 3}
    T = sum(_spread(case["B"], 1, case["new"]))
    return {"bytes": 2 * T * (Hq + 2 * Hk) * D * e, "flops": T * (Hq + Hk) * ops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        for pool in s["pools"]:                       # a copy: the values themselves
            for a, b in zip(s["src"], s["dst"]):
                pool[b].copy_(pool[a])
        return s["pools"]
    with torch.no_grad():
        return _exact_attend(s) if case["op"] == "attend" else _exact_rotary(s)


def _exact_attend(s):
    """softmax(q k / sqrt(D)) v over the last keys of each sequence, two passes in fp64, a key head at a time."""
    c = s["case"]
    B, Hq, Hk, D = c["B"], c["Hq"], c["Hk"], c["D"]
    out = torch.zeros(B, Hk, Hq // Hk, D, dtype=torch.float64, device="cuda")
    where = s["table"].long()
    for b in range(B):
        n = s["lengths"][b]
        lo = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            continue
        rows = torch.arange(lo, n, device="cuda")
        rows = where[b, rows // c["page"]] * c["page"] + rows % c["page"]
        for h in range(Hk):
            q = s["q"][b, h * (Hq // Hk):(h + 1) * (Hq // Hk)].double()
            k = s["k_pages"].view(-1, Hk, D)[rows, h].double()
            logits = torch.einsum("gd,nd->gn", q, k) / math.sqrt(D)
            del k
            weights = torch.softmax(logits, -1)
            v = s["v_pages"].view(-1, Hk, D)[rows, h].double()
            out[b, h] = torch.einsum("gn,nd->gd", weights, v)
    return out.view(B, Hq, D)


def _exact_rotary(s):
    """R(n(x)): n(x) = w x / r with r = sqrt(mean x^2 + eps), R the rotation of each pair as a product of complex numbers;
    and, for a step of training, dx = (w g - (x / r) mean(w g x / r)) / r and dw = sum g x / r with g = R^T dy."""
    c = s["case"]
    rot, D = c["rot"], c["D"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[..., None, None] * s["inv_freq"])
    even = torch.arange(0, rot, 2, device="cuda") if c["interleaved"] else torch.arange(rot // 2, device="cuda")
    odd = even + 1 if c["interleaved"] else even + rot // 2

    def rotate(x, by):
        z = torch.complex(x[..., even], x[..., odd]) * by
        y = x.clone()
        y[..., even], y[..., odd] = z.real, z.imag
        return y

    res, grads, dws = [], [], []
    for name in "qk":
        x, w = s[name].double(), s["w" + name]
        w = None if w is None else w.double()
        r = None if w is None else torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        res.append(rotate(x if w is None else x / r * w, turn))
        if c["op"] == "rotary" and c["train"]:
            g = rotate(s["d" + name].double(), turn.conj())
            if w is None:
                grads.append(g)
            else:
                u = x / r
                grads.append((w * g - u * (w * g * u).mean(-1, keepdim=True)) / r)
                dws.append((g * u).reshape(-1, D).sum(0))
    if c["op"] == "rotary":
        return (*res, *grads, *dws)
    rows = s["positions"].long()
    rows = s["table"].long()[s["seq_ids"].long(), rows // c["page"]] * c["page"] + rows % c["page"]
    k, v = s["k_pages"].double(), s["v_pages"].double()
    k.view(-1, c["Hk"], D)[rows] = res[1]
    v.view(-1, c["Hk"], D)[rows] = s["v"].double()
    return res[0], k, v
