"""The low-bit decode operators, as they are measured.

Three operators of one quantised attention block, over a paged cache in 8 bits:

``append``      q/k RMSNorm + rotation of the raw projections; q out in fp16, the new K and V into the cache as e4m3
                codes with one power-of-two scale for each 16 positions and kv head;
``attention``   grouped-query attention of the new rows (one a sequence, or several) over that cache;
``projection``  products with weights in 4 bits, with a scale (and a zero point) for each group of columns.

``run`` computes them in plain torch operations, or, where ``own`` is true, by the library's entry points.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 64    # positions of a page
BLOCK = 16   # positions that share a scale
EPS = 1e-5
THETA = 1e6


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one token of one sequence in the small model (8 q / 2 kv heads of 64): the launch counts
        {"name": "append step 1", "op": "append", "nq": 8, "nkv": 2, "hd": 64, "seqs": 1, "new_lo": 1, "new_hi": 1,
         "pos_lo": 700, "pos_hi": 700, "layers": 8, "norm": True},
        # one token each of the 256 sequences of batched decode (8 q / 2 kv heads of 96)
        {"name": "append step 256", "op": "append", "nq": 8, "nkv": 2, "hd": 96, "seqs": 256, "new_lo": 1, "new_hi": 1,
         "pos_lo": 16, "pos_hi": 2303, "layers": 1, "norm": True},
        # a pass over the prompts of a wide model without q/k norms, starting at odd places of pages
        {"name": "append prompts", "op": "append", "nq": 32, "nkv": 8, "hd": 128, "seqs": 11, "new_lo": 33,
         "new_hi": 1401, "pos_lo": 0, "pos_hi": 37, "layers": 1, "norm": False},
        # the first steps of one sequence in the small model
        {"name": "attend step 1 short", "op": "attention", "nq": 8, "nkv": 2, "hd": 64, "seqs": 1, "new_lo": 1,
         "new_hi": 1, "pos_lo": 130, "pos_hi": 130},
        # the 256 ragged sequences of batched decode
        {"name": "attend step 256", "op": "attention", "nq": 8, "nkv": 2, "hd": 96, "seqs": 256, "new_lo": 1,
         "new_hi": 1, "pos_lo": 16, "pos_hi": 2303},
        # one sequence alone with a long cache in a wide model
        {"name": "attend step 1 long", "op": "attention", "nq": 32, "nkv": 8, "hd": 128, "seqs": 1, "new_lo": 1,
         "new_hi": 1, "pos_lo": 32766, "pos_hi": 32766},
        # many long sequences: the largest cache
        {"name": "attend step 64 long", "op": "attention", "nq": 8, "nkv": 2, "hd": 96, "seqs": 64, "new_lo": 1,
         "new_hi": 1, "pos_lo": 14000, "pos_hi": 32766},
        # a few proposed tokens a sequence checked at once
        {"name": "attend proposals 32x5", "op": "attention", "nq": 8, "nkv": 2, "hd": 96, "seqs": 32, "new_lo": 3,
         "new_hi": 5, "pos_lo": 100, "pos_hi": 4000},
        # a stretch of long prompts over what is cached of them
        {"name": "attend prompts", "op": "attention", "nq": 8, "nkv": 2, "hd": 96, "seqs": 4, "new_lo": 300,
         "new_hi": 512, "pos_lo": 0, "pos_hi": 4000},
        # the output projection of the 768-wide model for one token: the launch counts
        {"name": "project 768x768 b1", "op": "projection", "n": 768, "k": 768, "batch": 1, "group": 32,
         "zeros": False},
        # a large matrix for one token: the weights' bytes count
        {"name": "project 16384x8192 b1", "op": "projection", "n": 16384, "k": 8192, "batch": 1, "group": 128,
         "zeros": False},
        # a large matrix with zero points for a batch of sequences
        {"name": "project 8192x8192 b24", "op": "projection", "n": 8192, "k": 8192, "batch": 24, "group": 64,
         "zeros": True},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["append", "attention", "attention", "projection", "projection"])
    if op == "projection":
        group = rng.choice([32, 64, 128])
        k = group * log(1, 16384 // group)
        n = log(1, 16384)
        while n * k > 16384 * 8192:
            n = log(1, 16384)
        return {"op": op, "n": n, "k": k, "batch": log(1, 64), "group": group, "zeros": rng.random() < 0.5}
    nkv = rng.choice([1, 2, 3, 4, 8])
    rep = rng.choice([1, 2, 3, 4, 5, 7, 8])
    hd = rng.choice([16, 32, 64, 64, 96, 96, 128])
    case = {"op": op, "nq": nkv * rep, "nkv": nkv, "hd": hd}
    if op == "append":
        seqs = log(1, 256)
        hi = log(1, max(1, min(1401, 8000 // seqs)))
        layers = rng.choice([1, 2, 3])
        pos = log(1, min(2303, 200_000_000 // (seqs * layers * nkv * hd)))
        return {**case, "seqs": seqs, "new_lo": rng.randint(1, hi), "new_hi": hi, "pos_lo": rng.randint(0, pos),
                "pos_hi": pos, "layers": layers, "norm": rng.random() < 0.7}
    kind = rng.choice(["step", "step", "several", "prompts"])
    seqs = {"step": log(1, 256), "several": log(1, 64), "prompts": log(1, 4)}[kind]
    hi = {"step": 1, "several": rng.randint(2, 8), "prompts": log(16, 512)}[kind]
    # no more than the listed cases' cache bytes and products
    most = min(32766, 450_000_000 // (seqs * nkv * hd * 2), 8_000_000_000 // (seqs * hi * nkv * rep * hd * 4) + 16)
    pos = log(1, most)
    return {**case, "seqs": seqs, "new_lo": rng.randint(1, hi), "new_hi": hi, "pos_lo": rng.randint(0, pos),
            "pos_hi": pos}


def spread(lo, hi, n, step):
    """n whole numbers over [lo, hi], evenly, in an order that is not sorted (step: a prime above any n)."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * (i * step % n) // (n - 1) for i in range(n)]


def lengths(c):
    """Positions before the call and new rows of each sequence."""
    return spread(c["pos_lo"], c["pos_hi"], c["seqs"], 7919), spread(c["new_lo"], c["new_hi"], c["seqs"], 6841)


def work(c):
    if c["op"] == "projection":
        n, k, b = c["n"], c["k"], c["batch"]
        w = n * k / 2 + n * (k // c["group"]) * (3 if c["zeros"] else 2)
        return {"bytes": w + 2 * b * k + 4 * b * n, "flops": 2 * b * n * k}
    pos, new = lengths(c)
    rows = sum(new)
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    if c["op"] == "append":
        scales = sum(len({(p + i) // BLOCK for i in range(m)}) for p, m in zip(pos, new))
        io = 4 * rows * (nq + 2 * nkv) * hd + 2 * rows * nq * hd
        return {"bytes": io + 2 * rows * nkv * hd + 8 * scales * nkv + 4 * rows * hd,
                "flops": 8 * rows * (nq + nkv) * hd}
    cached = sum(p + m for p, m in zip(pos, new))
    pairs = sum(m * p + m * (m + 1) // 2 for p, m in zip(pos, new))
    return {"bytes": 2 * cached * nkv * (hd + 4 / BLOCK) + 4 * rows * nq * hd, "flops": 4 * pairs * nq * hd}


# ------------------------------------------------------------------ inputs

def pow2_scale(amax):
    """The smallest power of two s with amax <= 448 s (448: the largest e4m3 value)."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.full_like(amax, 2.0 ** -126))


def random_cache(g, n_pages, layers, nkv, hd):
    """A pool whose every position holds a value, as stale ones do after use: K near unit norm, V of another size in
    each head, both with a few larger channels."""
    x = torch.randn(n_pages, layers, 2, nkv, PAGE // BLOCK, BLOCK, hd, device="cuda", generator=g)
    size = torch.exp(0.7 * torch.randn(2, nkv, 1, 1, hd, device="cuda", generator=g))
    x *= size / size.square().mean(-1, keepdim=True).sqrt()
    x[:, :, 1] *= 0.25
    s = pow2_scale(x.abs().amax((-1, -2)))
    x /= s[..., None, None]
    codes = x.to(torch.float8_e4m3fn).view(torch.uint8).reshape(n_pages, layers, 2, nkv, PAGE, hd)
    return codes.contiguous(), s.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = case
    st = {"case": c}
    if c["op"] == "projection":
        n, k, b, group = c["n"], c["k"], c["batch"], c["group"]
        st["codes"] = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
        sc = 0.006 * torch.exp(0.3 * torch.randn(n, k // group, device="cuda", generator=g))
        st["scales"] = sc.half()
        st["zeros"] = (torch.randint(5, 11, (n, k // group), dtype=torch.uint8, device="cuda", generator=g)
                       if c["zeros"] else None)
        x = torch.randn(b, k, device="cuda", generator=g)
        st["x"] = (x * torch.exp(0.5 * torch.randn(k, device="cuda", generator=g))).half()
        st["y"] = torch.empty(b, n, device="cuda")
        return st
    pos, new = lengths(c)
    seqs, nq, nkv, hd = c["seqs"], c["nq"], c["nkv"], c["hd"]
    layers = c.get("layers", 1)
    need = [-(-(p + m) // PAGE) for p, m in zip(pos, new)]
    n_pages, max_pages, max_seqs = sum(need) + 3, max(need), seqs + 2
    at = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    slots = torch.randperm(max_seqs, device="cuda", generator=g)[:seqs].to(torch.int32)
    needs = torch.tensor(need, device="cuda")
    begin = torch.cumsum(needs, 0) - needs
    col = torch.arange(max_pages, device="cuda")
    own_page = at[(begin[:, None] + col).clamp(max=n_pages - 1)]
    table = torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device="cuda")
    table[slots.long()] = torch.where(col < needs[:, None], own_page, -1)
    seq_pos = torch.zeros(max_seqs, dtype=torch.int32, device="cuda")
    seq_pos[slots.long()] = torch.tensor(pos, dtype=torch.int32, device="cuda")
    start = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
    start[1:] = torch.cumsum(torch.tensor(new, device="cuda"), 0)
    rows = sum(new)
    codes, scales = random_cache(g, n_pages, layers, nkv, hd)
    st.update(layer=layers - 1, layers=layers, rows=rows, max_new=max(new), max_ctx=max(p + m for p, m in zip(pos, new)),
              n_pages=n_pages, max_pages=max_pages, max_seqs=max_seqs, table=table, seq_pos=seq_pos, slots=slots,
              start=start, codes=codes, scales=scales, error=torch.zeros(1, dtype=torch.int32, device="cuda"))
    if c["op"] == "append":
        max_pos = max(p + m for p, m in zip(pos, new))
        ang = torch.arange(max_pos, device="cuda", dtype=torch.float64)[:, None] * (
            THETA ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) * 2 / hd))
        st.update(max_pos=max_pos, cos=ang.cos().float().contiguous(), sin=ang.sin().float().contiguous(),
                  qkv=torch.randn(rows, (nq + 2 * nkv) * hd, device="cuda", generator=g),
                  q_norm=1 + 0.2 * torch.randn(hd, device="cuda", generator=g) if c["norm"] else None,
                  k_norm=1 + 0.2 * torch.randn(hd, device="cuda", generator=g) if c["norm"] else None,
                  q=torch.empty(rows, nq * hd, dtype=torch.float16, device="cuda"))
    else:
        st.update(q=(1.7 * torch.randn(rows, nq * hd, device="cuda", generator=g)).half(),
                  out=torch.empty(rows, nq * hd, dtype=torch.float16, device="cuda"))
    return st


# ------------------------------------------------------------------ plain forms

def plain_append(st):
    c = st["case"]
    nq, nkv, hd, lay = c["nq"], c["nkv"], c["hd"], st["layer"]
    rows, half = st["rows"], hd // 2
    start, slots = st["start"].long(), st["slots"].long()
    r = torch.arange(rows, device="cuda")
    seq = torch.bucketize(r, start[1:], right=True)
    pos = st["seq_pos"].long()[slots[seq]] + r - start[seq]
    x = st["qkv"].view(rows, nq + 2 * nkv, hd)
    qk, v = x[:, :nq + nkv], x[:, nq + nkv:]
    if st["q_norm"] is not None:
        w = torch.cat([st["q_norm"].expand(nq, hd), st["k_norm"].expand(nkv, hd)])
        qk = qk / torch.sqrt(qk.square().mean(-1, keepdim=True) + EPS) * w
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    a, b = qk[..., :half], qk[..., half:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    q = qk[:, :nq].reshape(rows, nq * hd).half()
    kv = torch.stack([qk[:, nq:], v], 1)                                   # [rows][2][nkv][hd]

    # physical block of each row; its largest new value; whether older positions stay in it
    codes, scales = st["codes"][:, lay], st["scales"][:, lay]              # [page][2][nkv][64][hd], [page][2][nkv][4]
    n_blocks = st["n_pages"] * (PAGE // BLOCK)
    blk = st["table"].long()[slots[seq], pos // PAGE] * (PAGE // BLOCK) + pos % PAGE // BLOCK
    amax = torch.zeros(n_blocks, 2, nkv, device="cuda").index_reduce_(0, blk, kv.abs().amax(-1), "amax")
    first = blk[start[:-1]]
    offset = st["seq_pos"].long()[slots] % BLOCK
    kept = torch.zeros(n_blocks, dtype=torch.bool, device="cuda").index_put_((first,), offset > 0)
    touched = torch.zeros(n_blocks, dtype=torch.bool, device="cuda").index_put_((blk,), torch.tensor(True, device="cuda"))
    old = scales.permute(0, 3, 1, 2).reshape(n_blocks, 2, nkv)
    fresh = pow2_scale(amax)
    s = torch.where(kept[:, None, None], torch.maximum(old, fresh), fresh)
    s = torch.where(touched[:, None, None], s, old)

    # older positions of a first block go over to its new scale
    t = torch.arange(BLOCK, device="cuda")
    page, row0 = first // (PAGE // BLOCK), first % (PAGE // BLOCK) * BLOCK
    where = (page[:, None], slice(None), slice(None), row0[:, None] + t)    # [seqs][16][2][nkv][hd]
    was = codes[where].view(torch.float8_e4m3fn).float()
    again = was * (old[first] / s[first])[:, None, :, :, None]
    stays = (t < offset[:, None])[:, :, None, None, None]
    codes[where] = torch.where(stays, again.to(torch.float8_e4m3fn).view(torch.uint8), codes[where])

    new = (kv / s[blk][..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    codes[blk // (PAGE // BLOCK), :, :, pos % PAGE] = new
    scales.copy_(s.view(st["n_pages"], PAGE // BLOCK, 2, nkv).permute(0, 2, 3, 1))
    return {"q": q, "codes": st["codes"].view(torch.float8_e4m3fn), "scales": st["scales"]}


def plain_attention(st):
    c = st["case"]
    seqs, nq, nkv, hd, lay = c["seqs"], c["nq"], c["nkv"], c["hd"], st["layer"]
    rep, rows, new, ctx = nq // nkv, st["rows"], st["max_new"], st["max_ctx"]
    start, slots = st["start"].long(), st["slots"].long()
    pages = st["table"].long()[slots].clamp(min=0)                          # [seqs][max_pages]
    pos = st["seq_pos"].long()[slots]
    length = pos + start[1:] - start[:-1]
    t = torch.arange(pages.shape[1] * PAGE, device="cuda")

    def cached(which):
        x = st["codes"][pages, lay, which].view(torch.float8_e4m3fn).float()   # [seqs][pages][nkv][64][hd]
        s = st["scales"][pages, lay, which].repeat_interleave(BLOCK, -1, output_size=PAGE)
        x = (x * s[..., None]).transpose(1, 2).reshape(seqs, nkv, -1, hd)
        return x.masked_fill_((t >= length[:, None])[:, None, :, None], 0)[:, :, :ctx]

    i = torch.arange(new, device="cuda")
    at = (start[:-1, None] + i).clamp(max=rows - 1)                         # row of each (sequence, new token)
    q = st["q"].float().view(rows, nkv, rep, hd)[at].transpose(1, 2).reshape(seqs, nkv, new * rep, hd)
    score = (q @ cached(0).transpose(-1, -2)).view(seqs, nkv, new, rep, ctx) / math.sqrt(hd)
    hidden = t[:ctx] > (pos[:, None] + i)[..., None]                        # [seqs][new][ctx]
    score.masked_fill_(hidden[:, None, :, None], float("-inf"))
    score -= score.amax(-1, keepdim=True)
    p = score.exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(seqs, nkv, new * rep, ctx) @ cached(1)).view(seqs, nkv, new, rep, hd) / total
    r = torch.arange(rows, device="cuda")
    seq = torch.bucketize(r, start[1:], right=True)
    return out.transpose(1, 2)[seq, r - start[seq]].reshape(rows, nq * hd).half()


def plain_projection(st):
    c = st["case"]
    n, k, group = c["n"], c["k"], c["group"]
    codes = st["codes"]
    w = torch.stack([codes & 15, codes >> 4], -1).view(n, k // group, group).float()
    w -= 8.0 if st["zeros"] is None else st["zeros"].float()[..., None]
    w *= st["scales"].float()[..., None]
    return st["x"].float() @ w.view(n, k).t()


# ------------------------------------------------------------------ the library's operators

def ptr(t):
    return None if t is None else t.data_ptr()


def own_cache(st):
    from minimind_orangepi_b200._lib import Kv8Cache
    c = st["case"]
    return Kv8Cache(st["n_pages"], st["layers"], c["nkv"], c["hd"], st["max_seqs"], st["max_pages"], ptr(st["codes"]),
                    ptr(st["scales"]), ptr(st["table"]), ptr(st["seq_pos"]), ptr(st["error"]))


def own_append(st):
    from minimind_orangepi_b200._lib import check, lib
    c = st["case"]
    check(lib().mmc_op_kv8_append(own_cache(st), st["layer"], c["seqs"], st["rows"], st["max_new"], ptr(st["slots"]),
                                  ptr(st["start"]), c["nq"], ptr(st["qkv"]), ptr(st["q_norm"]), ptr(st["k_norm"]),
                                  ptr(st["cos"]), ptr(st["sin"]), st["max_pos"], EPS, ptr(st["q"]),
                                  torch.cuda.current_stream().cuda_stream))
    return {"q": st["q"], "codes": st["codes"].view(torch.float8_e4m3fn), "scales": st["scales"]}


def own_attention(st):
    import ctypes

    from minimind_orangepi_b200._lib import check, lib
    c = st["case"]
    cache = own_cache(st)
    if "ws" not in st:  # a program keeps its workspace
        size = ctypes.c_size_t()
        check(lib().mmc_op_kv8_attention_workspace_size(cache, c["seqs"], st["rows"], st["max_new"], c["nq"],
                                                        st["max_ctx"], ctypes.byref(size)))
        st["ws"] = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    check(lib().mmc_op_kv8_attention(cache, st["layer"], c["seqs"], st["rows"], st["max_new"], ptr(st["slots"]),
                                     ptr(st["start"]), c["nq"], ptr(st["q"]), st["max_ctx"], ptr(st["out"]),
                                     ptr(st["ws"]), st["ws"].numel(), torch.cuda.current_stream().cuda_stream))
    return st["out"]


def own_projection(st):
    from minimind_orangepi_b200._lib import check, lib
    c = st["case"]
    check(lib().mmc_op_w4_projection(c["batch"], c["n"], c["k"], c["group"], ptr(st["codes"]), ptr(st["scales"]),
                                     ptr(st["zeros"]), ptr(st["x"]), ptr(st["y"]),
                                     torch.cuda.current_stream().cuda_stream))
    return st["y"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": own_append, "attention": own_attention, "projection": own_projection}[op](state)
    return {"append": plain_append, "attention": plain_attention, "projection": plain_projection}[op](state)


# ------------------------------------------------------------------ 64 bits, sequence by sequence

def exact_round_e4m3(x):
    """x to the nearest e4m3 value (ties to even), as float64: steps of 2^(e-3), e from -6 on."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact_scale(amax):
    e = torch.ceil(torch.log2(amax.clamp(min=1e-30) / 448.0))
    e = torch.where(torch.exp2(e - 1) * 448.0 >= amax, e - 1, e)
    e = torch.where(torch.exp2(e) * 448.0 < amax, e + 1, e)
    return torch.exp2(e.clamp(min=-126))


def exact_append(st):
    c = st["case"]
    nq, nkv, hd, lay = c["nq"], c["nkv"], c["hd"], st["layer"]
    pos, new = lengths(c)
    codes = st["codes"].view(torch.float8_e4m3fn).double()
    scales = st["scales"].double()
    table, slots = st["table"].tolist(), st["slots"].tolist()
    out = torch.empty(st["rows"], nq, hd, dtype=torch.float64, device="cuda")
    row = 0
    for s in range(c["seqs"]):
        p0, m = pos[s], new[s]
        x = st["qkv"][row:row + m].double().view(m, nq + 2 * nkv, hd)
        turned = []
        for lo, hi, w in ((0, nq, st["q_norm"]), (nq, nq + nkv, st["k_norm"])):
            y = x[:, lo:hi]
            if w is not None:
                y = y * torch.rsqrt((y * y).sum(-1, keepdim=True) / hd + EPS) * w.double()
            z = torch.complex(y[..., :hd // 2].contiguous(), y[..., hd // 2:].contiguous())
            turn = torch.complex(st["cos"][p0:p0 + m].double(), st["sin"][p0:p0 + m].double())[:, None]
            z = z * turn
            turned.append(torch.cat([z.real, z.imag], -1))
        out[row:row + m] = turned[0]
        kv = torch.stack([turned[1], x[:, nq + nkv:]], 0).permute(0, 2, 1, 3)   # [2][nkv][m][hd]
        p = p0
        while p < p0 + m:
            lo = p // BLOCK * BLOCK
            hi = min(lo + BLOCK, p0 + m)
            page, b, o = table[slots[s]][lo // PAGE], lo % PAGE // BLOCK, lo % PAGE
            fresh = kv[:, :, p - p0:hi - p0]
            size = exact_scale(fresh.abs().amax((-1, -2)))
            if p > lo:
                had = scales[page, lay, :, :, b].clone()
                size = torch.maximum(size, had)
                older = codes[page, lay, :, :, o:o + p - lo] * (had / size)[..., None, None]
                codes[page, lay, :, :, o:o + p - lo] = exact_round_e4m3(older)
            codes[page, lay, :, :, o + p - lo:o + hi - lo] = exact_round_e4m3(fresh / size[..., None, None])
            scales[page, lay, :, :, b] = size
            p = hi
        row += m
    return {"q": out.view(st["rows"], nq * hd), "codes": codes, "scales": scales}


def exact_attention(st):
    c = st["case"]
    nq, nkv, hd, lay = c["nq"], c["nkv"], c["hd"], st["layer"]
    pos, new = lengths(c)
    table, slots = st["table"].long(), st["slots"].tolist()
    out = torch.empty(st["rows"], nq, hd, dtype=torch.float64, device="cuda")
    row = 0
    for s in range(c["seqs"]):
        n, m = pos[s] + new[s], new[s]
        pages = table[slots[s], :-(-n // PAGE)]
        kv = st["codes"][pages, lay].view(torch.float8_e4m3fn).double().unflatten(3, (PAGE // BLOCK, BLOCK))
        kv = kv * st["scales"][pages, lay].double()[..., None, None]
        kv = kv.permute(1, 2, 0, 3, 4, 5).reshape(2, nkv, -1, hd)[:, :, :n]
        q = st["q"][row:row + m].double().view(m, nq, hd)
        seen = torch.ones(m, n, dtype=torch.bool, device="cuda").tril(n - m)
        for h in range(nq):
            w = q[:, h] @ kv[0, h * nkv // nq].T / math.sqrt(hd)
            w = torch.softmax(w.masked_fill(~seen, float("-inf")), -1)
            out[row:row + m, h] = w @ kv[1, h * nkv // nq]
        row += m
    return out.view(st["rows"], nq * hd)


def exact_projection(st):
    c = st["case"]
    n, k, group = c["n"], c["k"], c["group"]
    w = torch.empty(n, k, dtype=torch.float64, device="cuda")
    w[:, 0::2] = st["codes"] % 16
    w[:, 1::2] = st["codes"] // 16
    z = st["zeros"].double().repeat_interleave(group, 1) if st["zeros"] is not None else 8
    w = (w - z) * st["scales"].double().repeat_interleave(group, 1)
    return st["x"].double() @ w.T


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": exact_append, "attention": exact_attention, "projection": exact_projection}[case["op"]](st)
