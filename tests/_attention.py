"""Plain 64-bit forms of the attention operators for the tests: rotary
positions, the 8-bit cache rows, attention row by row."""
import math

import torch

E4M3_MAX = 448.0
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}  # half the spacing of values just above 1


def rotate(x, table_rows, interleaved):
    """x [T, H, D] float64, table_rows [T, rot]: cosines then sines."""
    half = table_rows.shape[1] // 2
    y = x.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = table_rows[:, None, i].double(), table_rows[:, None, half + i].double()
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def exponents(x):
    """Smallest e with max|x| <= 448 * 2^e per row (at least -126), by counting."""
    top = x.abs().amax(-1)
    e = torch.full(top.shape, -126, dtype=torch.int64, device=x.device)
    for k in range(-126, 121):
        e = torch.where(top > E4M3_MAX * 2.0 ** k, torch.full_like(e, k + 1), e)
    return e


def e4m3_grid(device):
    m, e = torch.meshgrid(torch.arange(8.), torch.arange(16.), indexing="ij")
    g = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7))
    return torch.sort(g.flatten()[g.flatten() <= E4M3_MAX]).values.double().to(device)


def nearest(y, grid):
    """(nearest grid value of |y| up to the largest, distance to the next rounding boundary relative to the step)."""
    a = y.abs().clamp(max=E4M3_MAX)
    hi = torch.searchsorted(grid, a).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi], grid[lo]
    value = torch.where(a - down < up - a, down, up)
    margin = ((a - (up + down) / 2).abs() / (up - down).clamp(min=1e-300))
    return torch.copysign(value, y), margin


def attention(q, k, v, first_seen, scale):
    """q [n, Hq, D] float64 over k, v [m, Hkv, D]; row i sees the keys below
    first_seen + i (all of them if None).  Returns the output, the sum
    A = sum_j p_j |v_j|, the largest sum_d |q_d k_jd| * scale a row saw, and
    per row max_j p_j max|v_j| and the number of keys."""
    n, Hq, D = q.shape
    m, Hkv, _ = k.shape
    out, mass = torch.zeros_like(q), torch.zeros_like(q)
    size, peak = (torch.zeros(n, Hq, dtype=torch.float64, device=q.device) for _ in range(2))
    seen = torch.full((n,), m, device=q.device)
    if first_seen is not None:
        seen = (first_seen + torch.arange(n, device=q.device)).clamp(0, m)
    mask = torch.arange(m, device=q.device) < seen[:, None]
    for h in range(Hq):
        kh, vh = k[:, h // (Hq // Hkv)], v[:, h // (Hq // Hkv)]
        if m == 0:
            continue
        s = torch.where(mask, (q[:, h] @ kh.T) * scale, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        out[:, h], mass[:, h] = p @ vh, p @ vh.abs()
        size[:, h] = torch.where(mask, q[:, h].abs() @ kh.abs().T, 0.0).amax(-1) * scale
        peak[:, h] = (p * vh.abs().amax(-1)).amax(-1) * seen
    return out, mass, size, peak


def tolerance(dtype, mass, size, peak):
    """What an output may be off: the probabilities and the output are
    rounded to the activation type (half a step each, relative to the mass
    sum_j p_j |v_j|); a score's fp32 sum over D products is off by at most
    about 16 units of 2^-24 of the sum of their sizes, which moves every
    probability by as much; exp2 and the division by the sum add 2^-20; a
    probability below the 16-bit type's normal range is off by up to 2^-25 of
    the largest contribution (each key's)."""
    u = UNIT[dtype]
    return (2 * u + 2 * 2.0 ** -20 * size[..., None] + 2.0 ** -18) * mass + 2.0 ** -24 * peak[..., None] + 2.0 ** -24


def check(out, ref, mass, size, peak):
    assert torch.isfinite(out).all(), "a value is not finite"
    tol = tolerance(out.dtype, mass, size, peak)
    over = ((out.double() - ref).abs() / tol).max().item() if out.numel() else 0.0
    assert over <= 1.0, f"{over:.2f} times the tolerance"


def log2_spread(gen, shape, device="cuda"):
    return torch.exp2(torch.randint(-3, 4, shape, generator=gen, device=device).float())


def pages_of(lens, page, gen, spare=2, device="cuda"):
    """(block table int32, number of pages): every sequence's pages in a random order of a pool."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen, device=device).to(torch.int32)
    table = torch.full((len(lens), max(need + [1]) + 1), -7, dtype=torch.int32, device=device)  # no page past the end
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    return table, total


def gather(cache, exp, table, i, n):
    """Sequence i's first n cached rows as float64 [n, Hkv, D]."""
    page = cache.shape[2]
    ids = table[i, :-(-n // page)].long()
    x = cache[ids].double()
    if exp is not None:
        x = x * torch.exp2(exp[ids].double() - 127)[..., None]
    return x.permute(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[:n]


def scale_of(D):
    return 1.0 / math.sqrt(D)
