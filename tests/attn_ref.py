"""Plain float64 forms of the attention-layer operators, and bounds of the kernels' rounding errors.

Bounds are absolute, value by value.  The last rounding is off by at most half a step (``eps / 2`` of the value); what the
fp32 arithmetic in front of it may add is counted in units of u = 2^-24 of the magnitudes it works on."""
import torch

U = 2.0 ** -24


def rounding(y, dtype):
    """Half a step of ``dtype`` at y: eps / 2 of the value, and below the smallest normal number, where the steps stay what
    they are there, half of that step (fp16: values under 2^-14 lie 2^-24 apart, so a rounding is off by up to 2^-25)."""
    f = torch.finfo(dtype)
    return (f.eps / 2 * y.abs()).clamp(min=f.smallest_normal * f.eps / 2)


def norm_rotate(x, w, positions, inv_freq, interleaved, scale, eps):
    """x float64 [.., H, D] -> (y, magnitudes whose rounding y inherits)."""
    D, rot = x.shape[-1], 2 * inv_freq.numel()
    u = x
    if w is not None:
        u = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    angle = positions.double()[..., None, None] * inv_freq.double()
    c, s = angle.cos() * scale, angle.sin() * scale
    a, b = (u[..., 0:rot:2], u[..., 1:rot:2]) if interleaved else (u[..., :rot // 2], u[..., rot // 2:rot])
    ya, yb = a * c - b * s, a * s + b * c
    mag = scale * (a.abs() + b.abs())
    join = (lambda p, q: torch.stack([p, q], -1).flatten(-2)) if interleaved else (lambda p, q: torch.cat([p, q], -1))
    return torch.cat([join(ya, yb), u[..., rot:]], -1), torch.cat([join(mag, mag), u[..., rot:].abs()], -1)


def norm_rotate_bound(y, mag, dtype):
    # the angle as a float of half turns (pi / 2 u), sine and cosine (2 ulp = 4 u), two products and a sum (3 u), the norm: sum
    # of up to 512 squares over lanes and halves (at most 16 + 5 additions deep, half of it through the root: 11 u), root
    # (2 ulp = 4 u), two products (2 u): below 26 u
    return rounding(y, dtype) + 26 * U * mag


def norm_rotate_bwd(dy, x, w, positions, inv_freq, interleaved, scale, eps):
    """Formula of the gradients, float64: dx and dw (None without a weight), and their magnitudes."""
    g, gm = norm_rotate(dy, None, -positions, inv_freq, interleaved, scale, 0.0)
    if w is None:
        return g, None, gm, None
    r = torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    xh, w = x / r, w.double()
    dx = (w * g - xh * (w * g * xh).mean(-1, keepdim=True)) / r
    mag = (w.abs() * gm + xh.abs() * (w.abs() * gm * xh.abs()).mean(-1, keepdim=True)) / r
    D = x.shape[-1]
    return dx, (g * xh).reshape(-1, D).sum(0), mag, (gm * xh.abs()).reshape(-1, D)


def gather(pages, table, n):
    """The first n rows of a sequence: [n, H, D]."""
    size = pages.shape[1]
    at = torch.arange(n, device=pages.device)
    return pages[table.long()[at // size], at % size]


def attend(q, k_pages, v_pages, table, lengths, softmax_scale, window=0):
    """float64: out [B, Hq, D], lse [B, Hq], and a bound of the kernel's error in front of the last rounding."""
    B, Hq, D = q.shape
    Hk = k_pages.shape[2]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    lse = torch.full((B, Hq), float("-inf"), dtype=torch.float64, device=q.device)
    for b, n in enumerate(lengths):
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        row = torch.full((1,), b, device=q.device).expand(-(-n // k_pages.shape[1])) if table is None else table[b]
        k, v = (gather(t, row, n)[lo:].double().repeat_interleave(Hq // Hk, 1) for t in (k_pages, v_pages))
        qb = q[b].double() * softmax_scale
        s = torch.einsum("hd,nhd->hn", qb, k)
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("hn,nhd->hd", p, v)
        lse[b] = torch.logsumexp(s, -1)
        # a score: D products summed (2 u a step in the tensor cores), scaled, subtracted (|s| 4 u), exponential (2 ulp): an
        # error of a probability in both sums; the probability as head and remainder: a head of 8 bits towards zero leaves less
        # than 2^-7 of it, which is rounded to 8 bits (2^-9 of it), so 2^-16; the sums over the keys of a warp, its lanes,
        # warps and blocks
        mag = torch.einsum("hd,nhd->hn", qb.abs(), k.abs()).amax(-1)
        c = 2 * ((2 * D + 8) * U * mag + 8 * U) + 2.0 ** -16 + 2 * U * (len(range(lo, n)) / 16 + 64)
        bound[b] = c[:, None] * torch.einsum("hn,nhd->hd", p, v.abs())
    return out, lse, bound
