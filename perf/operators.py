"""The attention operators next to the WLQ linears, as cases to be measured.

A decoder layer runs qkv projection -> rotary positions and cache write ->
attention -> o projection.  The projections are the WLQ linears; the cases
here are what stands between them when a model is served:

* ``cache``   rotary positions on q and k, k and v stored in a paged cache
  (16-bit values, or e4m3 codes with a power-of-two scale per token and head;
  an 8-bit cache is read back, so its contents come out as the values they
  stand for);
* ``read``    the cached k and v of whole sequences, read back as 16-bit rows;
* ``prompt``  causal attention of packed prompts of different lengths over
  their own k and v;
* ``paged``   causal attention of each sequence's newest tokens (one, or a
  chunk) over the paged cache.

``own`` false computes them in elementary torch operations in 32 bits, true
calls this package's kernels.  Page layout: caches [pages, kv_heads,
page_size, dim], scales uint8 [pages, kv_heads, page_size] (exponent + 127),
``block_table`` int32 [sequences, pages per sequence].
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
E4M3_MAX = 448.0


# ------------------------------------------------------------------ cases ---

def listed():
    big = {"heads": 28, "kv_heads": 4, "dim": 128, "dtype": "bf16"}    # a 7B model's attention
    small = {"heads": 14, "kv_heads": 2, "dim": 64, "dtype": "f16"}    # a 0.5B model's attention
    return [
        # one decoding step of 32 sequences: the smallest call of a layer, latency counts
        {"name": "cache step 32", "op": "cache", "batch": 32, "short": 1024, "long": 1280, "new": 1, "page": 16,
         "bits": 8, "rot": 128, "interleaved": False, "stretch": 1.0, **big},
        # an odd prompt into a 16-bit cache, neighbouring pairs, half of each head rotated
        {"name": "cache prompt 8191", "op": "cache", "batch": 1, "short": 8191, "long": 8191, "new": 8191, "page": 32,
         "bits": 16, "rot": 32, "interleaved": True, "stretch": 1.0, **small},
        # 32 prompts of 1024 tokens at once, positions scaled for long contexts
        {"name": "cache prompts 32x1024", "op": "cache", "batch": 32, "short": 1024, "long": 1024, "new": 1024,
         "page": 16, "bits": 8, "rot": 128, "interleaved": False, "stretch": 4.0, **big},
        # one short sequence leaves the cache (moved to another pool)
        {"name": "read 997", "op": "read", "batch": 1, "short": 997, "long": 997, "page": 16, "bits": 8, **small},
        # a batch of long sequences read back for a pass over their whole context
        {"name": "read 32 to 16384", "op": "read", "batch": 32, "short": 1024, "long": 16384, "page": 16, "bits": 8,
         **big},
        # a few short prompts of very different lengths, one token among them
        {"name": "prompt 6 to 131", "op": "prompt", "batch": 6, "short": 1, "long": 131, **small},
        # a server's mixed prompt batch
        {"name": "prompt 16 to 2048", "op": "prompt", "batch": 16, "short": 65, "long": 2048, **big},
        # one long prompt
        {"name": "prompt 8192", "op": "prompt", "batch": 1, "short": 8192, "long": 8192, **big},
        # one user's single token: latency
        {"name": "paged one 1501", "op": "paged", "batch": 1, "short": 1501, "long": 1501, "new": 1, "page": 16,
         "bits": 16, **big},
        # the batch of a server in steady decoding
        {"name": "paged 32 at 1280", "op": "paged", "batch": 32, "short": 1024, "long": 1280, "new": 1, "page": 16,
         "bits": 8, **big},
        # long contexts of very different lengths
        {"name": "paged 16 to 65536", "op": "paged", "batch": 16, "short": 2001, "long": 65536, "new": 1, "page": 16,
         "bits": 8, **big},
        # chunked prompts: 512 new tokens each over what is cached already
        {"name": "paged chunk 512", "op": "paged", "batch": 4, "short": 1501, "long": 16384, "new": 512, "page": 16,
         "bits": 8, **big},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads, kv_heads, dim = rng.choice([(28, 4, 128), (14, 2, 64), (32, 8, 128), (16, 16, 64), (8, 1, 128), (12, 2, 128),
                                       (10, 5, 64)])
    case = {"op": rng.choice(["cache", "read", "prompt", "paged", "paged"]), "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": rng.choice(["bf16", "f16"])}
    if case["op"] == "prompt":
        long = _log(rng, 16, 4000)
        most = max(1, int(1.0e9 / (heads * long * long)))
        case.update(batch=_log(rng, 1, min(48, most)), short=_log(rng, 1, long), long=long)
        return case
    case.update(page=rng.choice([16, 32, 64, 128]), bits=rng.choice([8, 8, 16]))
    kv = kv_heads * dim  # values of one token's k
    if case["op"] == "cache":
        batch = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, min(4000, 30000 // batch)))
        long = new + _log(rng, 1, 2000)
        case.update(batch=batch, new=new, short=_log(rng, new, long), long=long, rot=rng.choice([dim, dim, dim // 2]),
                    interleaved=rng.random() < 0.5, stretch=rng.choice([1.0, 4.0]))
    elif case["op"] == "read":
        long = _log(rng, 1, 20000)
        case.update(batch=_log(rng, 1, max(1, min(64, int(1.0e8 / (long * kv))))), short=_log(rng, 1, long), long=long)
    elif rng.random() < 0.6:  # single tokens
        long = _log(rng, 3, 60000)
        case.update(batch=_log(rng, 1, max(1, min(96, int(4.0e8 / (long * kv))))), short=_log(rng, 1, long), long=long,
                    new=1)
    else:  # a chunk of new tokens
        new = _log(rng, 2, 1000)
        long = new + _log(rng, 1, 15000)
        most = max(1, int(8.0e8 / (heads * new * long)))
        case.update(batch=_log(rng, 1, min(32, most)), short=_log(rng, new, long), long=long, new=new)
    return case


def lengths(case):
    """Sequence lengths from short to long, evenly spread over their logarithm, in a mixed order."""
    b, lo, hi = case["batch"], case["short"], case["long"]
    if b == 1:
        return [hi]
    lens = [int(round(lo * (hi / lo) ** (i / (b - 1)))) for i in range(b)]
    random.Random(b * 7919 + hi).shuffle(lens)
    return lens


def news(case):
    """New tokens of each sequence: the case's number, fewer for every third sequence where it is a chunk."""
    n = case["new"]
    if case["op"] == "cache" or n == 1:
        return [min(n, length) for length in lengths(case)]
    return [min(length, n if i % 3 else max(1, n // 2 + 1)) for i, length in enumerate(lengths(case))]


def work(case):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    lens = lengths(case)
    row = 2 * d if case.get("bits", 16) == 16 else d + 1  # one token's k (or v) of one head in the cache
    if case["op"] == "cache":
        t = sum(news(case))
        n = t * (2 * 2 * h * d + 2 * kv * (2 * d + row) + 4 * case["rot"] + 16)
        if case["bits"] == 8:
            n += t * 2 * kv * (row + 2 * d)
        return {"bytes": n, "flops": 3 * t * (h + kv) * case["rot"]}
    if case["op"] == "read":
        return {"bytes": sum(lens) * 2 * kv * (row + 2 * d), "flops": 0}
    if case["op"] == "prompt":
        return {"bytes": sum(lens) * 2 * d * (2 * h + 2 * kv), "flops": 4 * d * h * sum(n * (n + 1) // 2 for n in lens)}
    new = news(case)
    seen = sum(n * length - n * (n - 1) // 2 for n, length in zip(new, lens))
    return {"bytes": sum(lens) * 2 * kv * row + sum(new) * 2 * 2 * h * d, "flops": 4 * d * h * seen}


# ---------------------------------------------------------------- inputs ---

def _randn(gen, shape, dtype):
    """Normal values, with a spread of scales over the tokens as activations have it."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return (x * torch.exp(0.5 * torch.randn(shape[:1] + (1,) * (len(shape) - 1), generator=gen, device="cuda"))).to(dtype)


def _cu(lens):
    return torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, h, kv, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    lens = lengths(case)
    s = dict(case, batch=len(lens), longest=max(lens), scale=d ** -0.5)
    if case["op"] == "prompt":
        # q, k and v are the parts of one projection's output
        t = sum(lens)
        qkv = _randn(gen, (t, (h + 2 * kv) * d), dtype)
        s["q"], s["k"], s["v"] = (x.view(t, -1, d) for x in qkv.split([h * d, kv * d, kv * d], dim=1))
        s["cu"] = _cu(lens)
        s["out"] = torch.empty(t, h, d, device="cuda", dtype=dtype)
        return s
    page = case["page"]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3  # a pool with a few pages to spare
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s["table"], s["lens"], s["cu"] = table, torch.tensor(lens, dtype=torch.int32, device="cuda"), _cu(lens)
    s["exp"] = None, None
    if case["op"] == "cache":
        stored = dtype if case["bits"] == 16 else torch.float8_e4m3fn
        s["cache"] = tuple(torch.zeros(pages, kv, page, d, device="cuda", dtype=stored) for _ in range(2))
        if case["bits"] == 8:
            s["exp"] = tuple(torch.full((pages, kv, page), 127, device="cuda", dtype=torch.uint8) for _ in range(2))
        new = news(case)
        t = sum(new)
        qkv = _randn(gen, (t, (h + 2 * kv) * d), dtype)
        s["q"], s["k"], s["v"] = (x.view(t, -1, d) for x in qkv.split([h * d, kv * d, kv * d], dim=1))
        s["positions"] = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lens, new)])
        seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(new, device="cuda"))
        s["slots"] = table[seq, s["positions"] // page].long() * page + s["positions"] % page
        freq = 1e6 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        angle = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None] / case["stretch"] * freq
        s["cos_sin"] = torch.cat((angle.cos(), angle.sin()), 1).float()
        s["q_out"] = torch.empty(t, h, d, device="cuda", dtype=dtype)
        if case["bits"] == 8:
            # what the step writes is read back: the sequences' newest pages, from their first token on
            s["first"] = [(n - m) // page for n, m in zip(lens, new)]
            count = [n - f * page for n, f in zip(lens, s["first"])]
            s["read_table"] = torch.stack([
                torch.nn.functional.pad(row[f:], (0, f)) for row, f in zip(table, s["first"])]).contiguous()
            s["read_cu"] = _cu(count)
            s["k_out"], s["v_out"] = (torch.empty(sum(count), kv, d, device="cuda", dtype=dtype) for _ in range(2))
            s["count"] = sum(count)
        return s
    cache = [_randn(gen, (pages, kv, page, d), dtype) for _ in range(2)]
    if case["bits"] == 8:
        cache, s["exp"] = zip(*(_quantise(x.float()) for x in cache))
    s["cache"] = tuple(cache)
    if case["op"] == "read":
        s["count"] = sum(lens)
        s["k_out"], s["v_out"] = (torch.empty(sum(lens), kv, d, device="cuda", dtype=dtype) for _ in range(2))
        return s
    new = news(case)
    s["q"] = _randn(gen, (sum(new), h, d), dtype)
    s["new"] = max(new)
    s["cu_q"] = None if s["new"] == 1 else _cu(new)
    s["out"] = torch.empty_like(s["q"])
    return s


# ----------------------------------------------------------- plain forms ---

def _quantise(x):
    """32-bit rows -> (e4m3 codes, exponent + 127), the smallest exponent e with max|x| <= 448 * 2^e."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = (e - 9 + (m > E4M3_MAX / 512)).clamp(-126, 127)
    code = (x * torch.exp2(-e[..., None].float())).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return code, (e + 127).to(torch.uint8)


def _values(cache, exp):
    """A cache's contents as 32-bit values."""
    x = cache.float()
    return x if exp is None else x * torch.exp2(exp.float() - 127)[..., None]


def _sequences(cache, exp, table):
    """[sequences, kv_heads, pages * page_size, dim] 32-bit values of every sequence's pages."""
    x = _values(cache[table.long()], None if exp is None else exp[table.long()])
    return x.transpose(1, 2).flatten(2, 3)


def _rows(cu, count, longest):
    """(sequence, position) of each of `count` packed rows, and the [sequences, longest] row numbers of padded ones."""
    at = torch.arange(count, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), at, right=True)
    pad = (cu[:-1, None] + torch.arange(longest, device=cu.device)).clamp(max=count - 1)
    return seq, at - cu[seq], pad


def _attend(q, k, v, seen, scale):
    """q [b, kv, g, n, d] over k, v [b, kv, m, d]; seen [b, n, m] says which keys a row has. Rows without any give 0."""
    score = torch.matmul(q, k.transpose(-1, -2)[:, :, None]) * scale
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    return torch.matmul(p, v[:, :, None]) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_prompt(s):
    q, k, v = (s[n].float() for n in "qkv")
    count, (kv, d) = q.shape[0], k.shape[1:]
    seq, pos, pad = _rows(s["cu"], count, s["longest"])
    q = q.view(count, kv, -1, d)[pad].permute(0, 2, 3, 1, 4)
    k, v = (x[pad].transpose(1, 2) for x in (k, v))
    at = torch.arange(s["longest"], device="cuda")
    seen = (at <= at[:, None]).expand(s["batch"], -1, -1)
    out = _attend(q, k, v, seen, s["scale"])
    return out.permute(0, 3, 1, 2, 4)[seq, pos].flatten(1, 2).to(s["q"].dtype)


def _plain_paged(s):
    (k, v), q = (_sequences(c, e, s["table"]) for c, e in zip(s["cache"], s["exp"])), s["q"].float()
    count, kv, d = q.shape[0], k.shape[1], k.shape[3]
    cu = s["cu_q"] if s["cu_q"] is not None else torch.arange(s["batch"] + 1, device="cuda", dtype=torch.int32)
    seq, pos, pad = _rows(cu, count, s["new"])
    q = q.view(count, kv, -1, d)[pad].permute(0, 2, 3, 1, 4)
    last = s["lens"] - (cu[1:] - cu[:-1])
    last = last[:, None] + torch.arange(s["new"], device="cuda")
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key <= last[..., None]) & (key < s["lens"][:, None, None])
    out = _attend(q, k, v, seen, s["scale"])
    return out.permute(0, 3, 1, 2, 4)[seq, pos].flatten(1, 2).to(s["q"].dtype)


def _rotate(x, cs, interleaved):
    half = cs.shape[1] // 2
    c, sn = cs[:, None, :half], cs[:, None, half:]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * c - b * sn, b * c + a * sn), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * c - b * sn, b * c + a * sn), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_read(s, table, cu):
    seq, pos, _ = _rows(cu, s["count"], 1)
    page = s["page"]
    slot = table[seq, pos // page].long()
    return [_values(c[slot, :, pos % page], None if e is None else e[slot, :, pos % page]).to(DTYPES[s["dtype"]])
            for c, e in zip(s["cache"], s["exp"])]


def _plain_cache(s):
    cs = s["cos_sin"][s["positions"]]
    q = _rotate(s["q"].float(), cs, s["interleaved"]).to(s["q"].dtype)
    k, v = _rotate(s["k"].float(), cs, s["interleaved"]), s["v"].float()
    page, off = s["slots"] // s["page"], s["slots"] % s["page"]
    for x, cache, exp in zip((k, v), s["cache"], s["exp"]):
        if exp is None:
            cache[page, :, off] = x.to(cache.dtype)
        else:
            code, e = _quantise(x)
            cache.view(torch.uint8)[page, :, off] = code.view(torch.uint8)
            exp[page, :, off] = e
    if s["bits"] == 8:
        return [q] + _plain_read(s, s["read_table"], s["read_cu"])
    return [q, *s["cache"]]


# ------------------------------------------------------------------- run ---

def run(s):
    if not own:
        if s["op"] == "cache":
            return _plain_cache(s)
        if s["op"] == "read":
            return _plain_read(s, s["table"], s["cu"])
        return _plain_prompt(s) if s["op"] == "prompt" else _plain_paged(s)
    from qwen_wlqfastshot_helen_beta_b200 import _C
    if s["op"] == "prompt":
        _C.prompt_attention(s["q"], s["k"], s["v"], s["cu"], s["out"], s["scale"])
        return s["out"]
    (k_cache, v_cache), (k_exp, v_exp) = s["cache"], s["exp"]
    if s["op"] == "paged":
        _C.paged_attention(s["q"], k_cache, v_cache, s["table"], s["lens"], s["out"], s["cu_q"], s["new"], k_exp, v_exp,
                           s["scale"])
        return s["out"]
    if s["op"] == "read":
        _C.kv_read(k_cache, v_cache, s["table"], s["cu"], s["k_out"], s["v_out"], k_exp, v_exp)
        return [s["k_out"], s["v_out"]]
    _C.rope_kv_write(s["q"], s["k"], s["v"], s["positions"], s["cos_sin"], s["slots"], k_cache, v_cache, s["q_out"],
                     None, k_exp, v_exp, s["interleaved"])
    if s["bits"] == 16:
        return [s["q_out"], k_cache, v_cache]
    _C.kv_read(k_cache, v_cache, s["read_table"], s["read_cu"], s["k_out"], s["v_out"], k_exp, v_exp)
    return [s["q_out"], s["k_out"], s["v_out"]]


# ----------------------------------------------------- 64-bit definitions ---

def _pow2(e):
    """2^e in 64 bits, exact (a library's power need not be)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_quantised(x):
    """The values that e4m3 codes with the row's power-of-two scale stand for, from the grid itself."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / E4M3_MAX)).clamp(-126, 127)
    y = x * _pow2(-e)
    binade = (y.abs().clamp(min=2.0 ** -6).view(torch.int64) >> 52) - 1023
    return torch.round(y * _pow2(3 - binade)).mul(_pow2(binade - 3)).clamp(-E4M3_MAX, E4M3_MAX) * _pow2(e)


def _exact_softmax(q, k, v, seen, scale):
    w = (q @ k.T) * scale
    w = torch.where(seen, w, torch.full_like(w, -math.inf))
    return torch.softmax(w, -1) @ v


def _exact_attention(q, keys, values, lens, new, scale):
    """Row by row of heads and sequences: q [t, h, d]; keys(i), values(i) give sequence i's [n, kv, d]."""
    out, at = torch.empty_like(q), 0
    for i, (n, m) in enumerate(zip(lens, new)):
        k, v = keys(i), values(i)
        group = q.shape[1] // k.shape[1]
        for h in range(q.shape[1]):
            for lo in range(0, m, 2048):
                hi = min(m, lo + 2048)
                seen = torch.arange(n, device="cuda") <= torch.arange(n - m + lo, n - m + hi, device="cuda")[:, None]
                out[at + lo:at + hi, h] = _exact_softmax(q[at + lo:at + hi, h], k[:, h // group], v[:, h // group],
                                                         seen, scale)
        at += m
    return out


def exact(case, seed):
    s = prepare(case, seed)
    lens, op = lengths(case), case["op"]

    def cached(which, i, n, table):
        c, e = s["cache"][which], s["exp"][which]
        page = table[i, :-(-n // s["page"])].long()
        x = c[page].double()
        if e is not None:
            x = x * _pow2(e[page].long() - 127)[..., None]
        return x.permute(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[:n]

    if op == "prompt":
        q, k, v = (s[n].double() for n in "qkv")
        cu = s["cu"].tolist()
        return _exact_attention(q, lambda i: k[cu[i]:cu[i + 1]], lambda i: v[cu[i]:cu[i + 1]], lens, lens, s["scale"])
    if op == "paged":
        return _exact_attention(s["q"].double(), lambda i: cached(0, i, lens[i], s["table"]),
                                lambda i: cached(1, i, lens[i], s["table"]), lens, news(case), s["scale"])
    if op == "read":
        return [torch.cat([cached(w, i, n, s["table"]) for i, n in enumerate(lens)]) for w in range(2)]
    # the angles are the 32-bit table's, which is an input
    turn = torch.complex(*s["cos_sin"].double()[s["positions"]].chunk(2, 1))[:, None]
    half = case["rot"] // 2

    def rotated(x):
        x = x.double()
        pair = x[..., :2 * half].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
        if not case["interleaved"]:
            pair = pair.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        if not case["interleaved"]:
            z = z.transpose(-1, -2)
        return torch.cat((z.reshape(*x.shape[:-1], 2 * half), x[..., 2 * half:]), -1)

    q, k, v = rotated(s["q"]), rotated(s["k"]), s["v"].double()
    if case["bits"] == 8:
        k, v = _exact_quantised(k), _exact_quantised(v)
    kv, d, page = case["kv_heads"], case["dim"], case["page"]
    pools = [c.double().transpose(1, 2).reshape(-1, kv, d) for c in s["cache"]]
    for pool, x in zip(pools, (k, v)):
        pool[s["slots"]] = x
    if case["bits"] == 16:
        return [q] + [p.view(-1, page, kv, d).transpose(1, 2) for p in pools]
    cu = s["read_cu"].tolist()
    slot = torch.cat([(s["read_table"][i].long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:b - a]
                      for i, (a, b) in enumerate(zip(cu, cu[1:]))])
    return [q] + [p[slot] for p in pools]
