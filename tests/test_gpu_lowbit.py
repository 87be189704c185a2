"""The low-bit operators against their 64-bit forms, through the C ABI: append and
attention over the 8-bit paged cache, 4-bit projections, and a run of them
together. The tolerances are derived where they are computed."""
from __future__ import annotations

import ctypes as C
import math
import os
import subprocess
import sys

import pytest

from minimind_orangepi_b200._lib import Kv8Cache, check, lib

torch = pytest.importorskip("torch")

from lowbit_reference import Cache, PAGE, attention, e4m3_table, norm_rope, w4_weights  # noqa: E402

pytestmark = pytest.mark.gpu

EPS = 1e-5
DEVICE_ERROR = 5


def ptr(t):
    return None if t is None else t.data_ptr()


class World:
    """A cache with random contents in every position, a table of shuffled pages, and the batch of one call."""

    def __init__(self, seed, nq, nkv, hd, pos, new, layers=1, layer=0, spare_rows=0, unused=(), size=1.0):
        g = self.g = torch.Generator().manual_seed(seed)
        self.nq, self.nkv, self.hd, self.layers, self.layer = nq, nkv, hd, layers, layer
        self.pos, self.new, self.seqs, self.unused = pos, new, len(pos), set(unused)
        need = [max(1, -(-(p + n) // PAGE)) for p, n in zip(pos, new)]
        self.n_pages, self.max_pages, self.max_seqs = sum(need) + 2, max(need) + 1, self.seqs + 2
        order = torch.randperm(self.n_pages, generator=g).tolist()
        self.slots = torch.randperm(self.max_seqs, generator=g)[:self.seqs].tolist()
        self.table = torch.full((self.max_seqs, self.max_pages), -1, dtype=torch.int32)
        self.seq_pos = torch.zeros(self.max_seqs, dtype=torch.int32)
        for i, s in enumerate(self.slots):
            for j in range(need[i]):
                self.table[s, j] = order.pop()
            self.seq_pos[s] = pos[i]
        self.start = [0]
        for n in new:
            self.start.append(self.start[-1] + n)
        self.rows = self.start[-1] + spare_rows
        self.codes = torch.randint(0, 256, (self.n_pages, layers, 2, nkv, PAGE, hd), dtype=torch.uint8, generator=g)
        # every byte, NaN codes too, where nothing is cached; e4m3 values with larger ones rare where something is
        x = (torch.randn(self.codes.shape, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
        x = x.view(torch.uint8)
        for i, s in enumerate(self.slots):
            for j in range(pos[i]):
                p = int(self.table[s, j // PAGE])
                self.codes[p, :, :, :, j % PAGE] = x[p, :, :, :, j % PAGE]
        e = torch.randint(-9, -5, (self.n_pages, layers, 2, nkv, PAGE // 16), generator=g)
        self.scales = torch.exp2(e.float()) * size
        self.device()

    def device(self):
        d = lambda t: t.cuda()  # noqa: E731
        self.d_codes, self.d_scales, self.d_table = d(self.codes), d(self.scales), d(self.table)
        self.d_pos = d(self.seq_pos)
        self.d_slots = d(torch.tensor([-1 if i in self.unused else s for i, s in enumerate(self.slots)],
                                      dtype=torch.int32))
        self.d_start = d(torch.tensor(self.start, dtype=torch.int32))
        self.d_err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.max_new = max(1, max(self.new))
        self.max_ctx = max(1, max(p + n for p, n in zip(self.pos, self.new)))
        self.cache = Kv8Cache(self.n_pages, self.layers, self.nkv, self.hd, self.max_seqs, self.max_pages,
                              ptr(self.d_codes), ptr(self.d_scales), ptr(self.d_table), ptr(self.d_pos),
                              ptr(self.d_err))
        half = self.hd // 2
        ang = torch.arange(self.max_ctx).double()[:, None] * 1e4 ** (-torch.arange(half).double() / half)
        self.cos, self.sin = ang.cos().float(), ang.sin().float()
        self.d_cos, self.d_sin = self.cos.cuda(), self.sin.cuda()

    def use_start(self):
        return None if self.rows == self.seqs and set(self.new) == {1} else ptr(self.d_start)

    def status(self):
        return lib().mmc_op_kv8_status(self.cache, None)

    def append(self, qkv, qn=None, kn=None, q=None, stream=None, start="auto"):
        q = torch.full((self.rows, self.nq * self.hd), 7.0, dtype=torch.float16, device="cuda") if q is None else q
        check(lib().mmc_op_kv8_append(self.cache, self.layer, self.seqs, self.rows, self.max_new, ptr(self.d_slots),
                                      self.use_start() if start == "auto" else start, self.nq, ptr(qkv), ptr(qn),
                                      ptr(kn), ptr(self.d_cos), ptr(self.d_sin), self.max_ctx, EPS, ptr(q), stream))
        return q

    def workspace(self, max_ctx=None):
        n = C.c_size_t()
        check(lib().mmc_op_kv8_attention_workspace_size(self.cache, self.seqs, self.rows, self.max_new, self.nq,
                                                        max_ctx or self.max_ctx, C.byref(n)))
        return torch.full((n.value,), 0xff, dtype=torch.uint8, device="cuda")  # NaN as floats

    def attend(self, q, out=None, ws=None, stream=None, max_ctx=None):
        out = torch.full((self.rows, self.nq * self.hd), 7.0, dtype=torch.float16, device="cuda") if out is None else out
        ws = self.workspace(max_ctx) if ws is None else ws
        check(lib().mmc_op_kv8_attention(self.cache, self.layer, self.seqs, self.rows, self.max_new, ptr(self.d_slots),
                                         self.use_start(), self.nq, ptr(q), max_ctx or self.max_ctx, ptr(out), ptr(ws),
                                         ws.numel(), stream))
        return out

    # ---- checks against the 64-bit forms
    def check_append(self, qkv, qn, kn, q):
        nq, nkv, hd, lay = self.nq, self.nkv, self.hd, self.layer
        ref = Cache(self.codes, self.scales)
        got_c = e4m3_table()[self.d_codes.cpu().long()]
        got_s = self.d_scales.cpu().double()
        x = qkv.cpu().view(self.rows, nq + 2 * nkv, hd)
        q = q.cpu().double().view(self.rows, nq, hd)
        for i in range(self.seqs):
            r0, r1, p0, n = self.start[i], self.start[i + 1], self.pos[i], self.new[i]
            if i in self.unused:
                assert (q[r0:r1] == 7).all()
                continue
            if n == 0:
                continue
            cos, sin = self.cos[p0:p0 + n, None], self.sin[p0:p0 + n, None]
            want = norm_rope(x[r0:r1, :nq], qn, cos, sin, EPS)
            # fp32: the norm's sum and factors and two products and a sum, each 2^-24 of the pair's size; fp16: half a step
            a, b = norm_rope(x[r0:r1, :nq], qn, torch.ones_like(cos), torch.zeros_like(sin), EPS).abs().chunk(2, -1)
            pair = torch.cat([a + b, a + b], -1)
            assert ((q[r0:r1] - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -25 + (hd + 16) * 2.0 ** -24 * pair).all()
            k = norm_rope(x[r0:r1, nq:nq + nkv], kn, cos, sin, EPS)
            ref.append(lay, self.table[self.slots[i]], p0, torch.stack([k, x[r0:r1, nq + nkv:].double()]).transpose(1, 2))
        live = ~got_s.isnan()
        assert torch.equal(live, ~ref.scales.isnan())
        assert torch.equal(got_s[live], ref.scales[live])
        # V has no arithmetic before its code: equal. K may fall on the other side of a border where fp32 and 64 bits
        # differ: by one step (an eighth of the value, 2^-9 at least), and seldom
        same = (got_c == ref.codes) | (got_c.isnan() & ref.codes.isnan())
        assert same[:, :, 1].all()
        diff = ~same[:, :, 0]
        assert diff.sum() <= max(2, 1e-3 * self.start[-1] * nkv * hd)
        g, w = got_c[:, :, 0][diff], ref.codes[:, :, 0][diff]
        assert ((g - w).abs() <= torch.maximum(w.abs(), g.abs()) / 8 + 2.0 ** -9).all()

    def check_attention(self, q, out, rows=None):
        ref = Cache(self.d_codes.cpu(), self.d_scales.cpu())
        q, out = q.cpu(), out.cpu().double()
        worst = 0.0
        for i in range(self.seqs):
            n = self.pos[i] + self.new[i]
            if self.new[i] == 0:
                continue
            r0 = self.start[i]
            if i in self.unused:
                assert (out[r0:r0 + self.new[i]] == 0).all()
                continue
            kv = ref.read(self.layer, self.table[self.slots[i]], n)
            for j in range(self.new[i]):
                want, tol = attention(q[r0 + j].view(self.nq, self.hd), kv, self.pos[i] + j)
                err = (out[r0 + j].view(self.nq, self.hd) - want).abs()
                assert (err <= tol).all(), (i, j, float((err / tol).max()))
                worst = max(worst, float((err / tol).max()))
        assert (out[self.start[-1]:] == 7).all()  # rows behind the last sequence
        return worst


def qkv_of(w, size=1.0):
    x = torch.randn(w.rows, (w.nq + 2 * w.nkv) * w.hd, generator=w.g) * size
    return x.cuda()


def q_of(w, size=1.5):
    return (torch.randn(w.rows, w.nq * w.hd, generator=w.g) * size).half().cuda()


def norms_of(w):
    return [(1 + 0.2 * torch.randn(w.hd, generator=w.g)) for _ in range(2)]


SHAPES = [(8, 2, 64), (8, 2, 96), (4, 4, 16), (6, 2, 32), (10, 2, 128), (7, 1, 96), (40, 2, 64), (3, 3, 128)]

# positions before the call, new rows
BATCHES = {
    "one": ([0], [1]),
    "steps": ([0, 1, 15, 16, 17, 63, 64, 65, 200, 511, 1000], [1] * 11),
    "several": ([0, 3, 14, 60, 129, 300], [2, 5, 3, 8, 0, 7]),
    "prompts": ([0, 5, 64, 0], [130, 75, 64, 1]),
}


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("nq,nkv,hd", SHAPES)
def test_append(nq, nkv, hd, batch):
    pos, new = BATCHES[batch]
    w = World(hd * 7 + nq, nq, nkv, hd, pos, new, layers=2, layer=1)
    x = qkv_of(w)
    qn, kn = norms_of(w) if nq != 7 else (None, None)
    q = w.append(x, qn.cuda() if qn is not None else None, kn.cuda() if kn is not None else None)
    assert w.status() == 0
    w.check_append(x, qn, kn, q)


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("nq,nkv,hd", SHAPES)
def test_attention(nq, nkv, hd, batch):
    pos, new = BATCHES[batch]
    w = World(hd * 9 + nq, nq, nkv, hd, pos, new, layers=2, layer=0)
    # the new positions hold values too: append before attending
    w.append(qkv_of(w))
    q = q_of(w)
    out = w.attend(q)
    assert w.status() == 0
    w.check_attention(q, out)


@pytest.mark.parametrize("nq,nkv,hd,pos,new", [
    (8, 2, 96, [8191], [1]), (8, 2, 64, [20000], [1]), (16, 8, 128, [5000, 0, 77], [1, 1, 1]),
    (8, 2, 96, [4000, 1500], [5, 33]), (8, 1, 32, [32700], [4]), (64, 1, 64, [900], [3])])
def test_attention_long(nq, nkv, hd, pos, new):
    w = World(sum(pos) + hd, nq, nkv, hd, pos, new)
    w.append(qkv_of(w))
    q = q_of(w)
    out = w.attend(q)
    assert w.status() == 0
    w.check_attention(q, out)


def test_attention_many_sequences():
    g = torch.Generator().manual_seed(11)
    pos = torch.randint(0, 700, (256,), generator=g).tolist()
    w = World(12, 8, 2, 96, pos, [1] * 256)
    w.append(qkv_of(w))
    q = q_of(w)
    out = w.attend(q)
    assert w.status() == 0
    w.check_attention(q, out)


def test_unused_rows_and_spare_rows():
    """A padded batch: unused sequences, rows behind the last one."""
    w = World(5, 8, 2, 64, [70, 10, 33, 5], [3, 2, 1, 4], spare_rows=5, unused=(1, 3))
    before = w.d_codes.clone(), w.d_scales.clone()
    x = qkv_of(w)
    q = w.append(x)
    assert w.status() == 0
    assert (q[w.start[-1]:] == 7).all()
    w.check_append(x, None, None, q)
    for i in (1, 3):
        pages = [p for p in w.table[w.slots[i]].tolist() if p >= 0]
        assert torch.equal(w.d_codes[pages], before[0][pages]) and torch.equal(w.d_scales[pages], before[1][pages])
    qq = q_of(w)
    out = w.attend(qq)
    assert w.status() == 0
    w.check_attention(qq, out)


def test_nothing_to_do():
    """Every sequence unused, or without rows."""
    w = World(6, 8, 2, 64, [70, 10], [1, 1], unused=(0, 1))
    out = w.attend(q_of(w))
    assert w.status() == 0 and (out == 0).all()
    w = World(7, 8, 2, 64, [70, 10], [0, 0], spare_rows=3)
    before = w.d_codes.clone()
    q = w.append(qkv_of(w))
    out = w.attend(q_of(w))
    assert w.status() == 0 and (out == 7).all() and (q == 7).all() and torch.equal(w.d_codes, before)


@pytest.mark.parametrize("hd", [16, 64, 96, 128])
def test_growing_scales_step_by_step(hd):
    """Tokens of growing, shrinking, zero and huge sizes, one a call: each step equals the 64-bit form applied to the
    cache that the step found, and the V codes equal those of one append of all of them (scales are powers of two; the
    sizes here keep every older code normal)."""
    n = 40
    size = [0.0, 1.0, 1.9, 0.5, 3.0, 8.0, 7.0, 20.0] * 5
    w = World(hd, 4, 2, hd, [0], [n])
    base = torch.randn(n, (w.nq + 2 * w.nkv) * hd, generator=w.g).sign() * (
        0.75 + 0.25 * torch.rand(n, (w.nq + 2 * w.nkv) * hd, generator=w.g))
    x = (base * torch.tensor(size)[:, None]).cuda()
    w.append(x)
    whole = w.d_codes.clone(), w.d_scales.clone()
    one = World(hd, 4, 2, hd, [0], [n])
    one.rows, one.max_new, one.new, one.start = 1, 1, [1], [0, 1]
    for i in range(n):
        one.codes, one.scales = one.d_codes.cpu(), one.d_scales.cpu()
        one.pos = [i]
        one.d_pos[one.slots[0]] = i
        row = x[i:i + 1].contiguous()
        q = one.append(row)
        assert one.status() == 0
        one.check_append(row, None, None, q)
    used = [int(p) for p in w.table[w.slots[0]] if p >= 0]
    t = e4m3_table()
    for tok in range(n):
        p, r = used[tok // PAGE], tok % PAGE
        a, b = t[whole[0][p, 0, 1, :, r].cpu().long()], t[one.d_codes[p, 0, 1, :, r].cpu().long()]
        assert torch.equal(a, b)
    assert torch.equal(whole[1][used][:, 0, 1, :, :2], one.d_scales[used][:, 0, 1, :, :2])


@pytest.mark.parametrize("amax", [448.0, 448.00003, 449.0, 3.4e38, 1.75 * 2.0 ** -126, 1e-40, 1e-45, 0.0])
def test_scale_borders(amax):
    w = World(3, 2, 2, 32, [3, 16], [2, 1])
    x = qkv_of(w, 0.1 * min(amax, 1e37))
    x[:, -w.nkv * w.hd:].clamp_(-amax, amax)
    x[0, -1] = amax
    x[2, -w.hd - 5] = -amax
    q = w.append(x)
    assert w.status() == 0
    if 1e-38 < amax < 1e37:  # (q and K pass through products that leave fp32's range elsewhere)
        w.check_append(x, None, None, q)
        return
    ref = Cache(w.codes, w.scales)
    v = x.cpu().view(w.rows, w.nq + 2 * w.nkv, w.hd)[:, -w.nkv:].double()
    for i in range(w.seqs):
        vi = v[w.start[i]:w.start[i + 1]].transpose(0, 1)
        ref.append(0, w.table[w.slots[i]], w.pos[i], torch.stack([vi, vi]))
    assert torch.equal(w.d_scales.cpu().double()[:, :, 1], ref.scales[:, :, 1])
    got = e4m3_table()[w.d_codes.cpu().long()][:, :, 1]
    assert ((got == ref.codes[:, :, 1]) | got.isnan()).all()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_infinite_values(bad):
    """A block with an infinity or a NaN has the scale NaN from then on; every row that reads it is NaN, no other."""
    w = World(8, 8, 2, 64, [20, 20], [2, 2])
    x = qkv_of(w)
    x[1, -3] = bad  # V of the last kv head, second row of sequence 0
    q = w.append(x)
    assert w.status() == 0
    w.check_append(x, None, None, q)
    qq = q_of(w)
    out = w.attend(qq).cpu().view(4, 2, -1)
    assert out[:2, 1].isnan().all() and not out[:2, 0].isnan().any() and not out[2:].isnan().any()
    # later positions of that block: its scale stays NaN, its older codes stay
    w2 = World(8, 8, 2, 64, [22, 22], [2, 2])
    w2.d_codes.copy_(w.d_codes)
    w2.d_scales.copy_(w.d_scales)
    w2.codes, w2.scales = w.d_codes.cpu(), w.d_scales.cpu()
    x = qkv_of(w2)
    q = w2.append(x)
    assert w2.status() == 0
    w2.check_append(x, None, None, q)
    assert w2.d_scales.isnan().sum() == 1


def test_infinite_value_ahead_of_a_row():
    """Rows that see no position of a lost block are not touched by it, though they share its tile."""
    for pos in (14, 62, 0):
        w = World(9, 8, 2, 96, [pos], [18])
        x = qkv_of(w)
        x[17, :] = math.nan  # q, K and V of the last row
        w.append(x)
        q = q_of(w)
        out = w.attend(q)
        assert w.status() == 0
        free = (pos + 17) // 16 * 16 - pos  # rows before the lost block
        ref = Cache(w.d_codes.cpu(), w.d_scales.cpu())
        kv = ref.read(0, w.table[w.slots[0]], pos + free) if free else None
        for j in range(free):
            want, tol = attention(q[j].cpu().view(w.nq, w.hd), kv, pos + j)
            assert ((out[j].cpu().double().view(w.nq, w.hd) - want).abs() <= tol).all()
        assert out[free:].isnan().all()


def test_attention_extreme_scores():
    """Scores of thousands, equal scores, rows whose largest score comes last, blocks of very different V sizes."""
    for size, qs in ((1.0, 60000.0), (1.0, 0.0), (2.0 ** -20, 300.0), (2.0 ** 20, 3.0)):
        w = World(21, 8, 2, 96, [700, 64], [1, 2], size=size)
        w.d_scales[:, :, 1] *= torch.exp2(torch.randint(-20, 20, w.d_scales[:, :, 1].shape, generator=w.g).float()).cuda()
        w.append(qkv_of(w, size))
        q = (torch.randn(w.rows, w.nq * w.hd, generator=w.g).clamp(-1, 1) * qs).half().cuda()
        out = w.attend(q)
        assert w.status() == 0
        ref = Cache(w.d_codes.cpu(), w.d_scales.cpu())
        for i in range(w.seqs):
            kv = ref.read(0, w.table[w.slots[i]], w.pos[i] + w.new[i])
            for j in range(w.new[i]):
                r = w.start[i] + j
                want, tol = attention(q[r].cpu().view(w.nq, w.hd), kv, w.pos[i] + j)
                got = out[r].cpu().double().view(w.nq, w.hd)
                top = want.abs() + tol >= 65519  # past fp16: infinite or the largest value
                assert ((got - want).abs()[~top] <= tol[~top]).all()


# A max_ctx with which a call of more than 32 rows a kv head counts as long runs, whatever its sequences' lengths
LONG = 1 << 17

LONG_RUNS = {
    "prompts": ([0, 5, 64, 0], [130, 75, 64, 1]),
    "ragged": ([600, 0, 3, 1000, 63], [40, 300, 0, 17, 129]),
    "cached": ([5000, 190], [60, 2]),
}


@pytest.mark.parametrize("batch", LONG_RUNS)
@pytest.mark.parametrize("nq,nkv,hd", SHAPES)
def test_long_runs(nq, nkv, hd, batch):
    pos, new = LONG_RUNS[batch]
    w = World(hd * 5 + nq, nq, nkv, hd, pos, new, layers=2, layer=1, spare_rows=3)
    w.append(qkv_of(w))
    q = q_of(w)
    out = w.attend(q, max_ctx=LONG)
    assert w.status() == 0
    w.check_attention(q, out)
    # and with the parts that the batch's own lengths ask for
    out = w.attend(q)
    assert w.status() == 0
    w.check_attention(q, out)


@pytest.mark.parametrize("nq,nkv,hd,seqs", [(16, 4, 64, 40), (16, 4, 96, 40), (8, 1, 128, 520), (8, 1, 32, 520)])
def test_long_runs_of_many_sequences(nq, nkv, hd, seqs):
    """As many tiles of rows as CTAs, and more than are listed by each."""
    g = torch.Generator().manual_seed(seqs + hd)
    pos = torch.randint(0, 200, (seqs,), generator=g).tolist()
    new = [40 if i % 37 == 5 else int(n) for i, n in enumerate(torch.randint(0, 3, (seqs,), generator=g))]
    w = World(hd + seqs, nq, nkv, hd, pos, new, unused=(2, 5, 30))
    w.append(qkv_of(w))
    q = q_of(w)
    out = w.attend(q, max_ctx=LONG)
    assert w.status() == 0
    w.check_attention(q, out)


@pytest.mark.parametrize("spread", [4, 20, 35])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_long_runs_extreme_scores_and_scales(hd, spread):
    """V's blocks up to 2^(2 spread) apart, scores of thousands and equal ones."""
    for size, qs in ((1.0, 60000.0), (1.0, 0.0), (2.0 ** -10, 300.0)):
        w = World(23 + spread, 8, 2, hd, [300, 64, 0], [12, 30, 20], size=size)
        w.append(qkv_of(w, size))
        e = torch.randint(-spread, spread, w.d_scales[:, :, 1].shape, generator=w.g).float().cuda()
        w.d_scales[:, :, 1] *= torch.exp2(e)
        q = (torch.randn(w.rows, w.nq * w.hd, generator=w.g).clamp(-1, 1) * qs).half().cuda()
        out = w.attend(q, max_ctx=LONG)
        assert w.status() == 0
        ref = Cache(w.d_codes.cpu(), w.d_scales.cpu())
        for i in range(w.seqs):
            kv = ref.read(0, w.table[w.slots[i]], w.pos[i] + w.new[i])
            for j in range(w.new[i]):
                r = w.start[i] + j
                want, tol = attention(q[r].cpu().view(w.nq, w.hd), kv, w.pos[i] + j)
                got = out[r].cpu().double().view(w.nq, w.hd)
                top = want.abs() + tol >= 65519  # past fp16: infinite or the largest value
                assert ((got - want).abs()[~top] <= tol[~top]).all()


@pytest.mark.parametrize("pos", [14, 62, 0])
def test_long_runs_infinite_value_ahead_of_a_row(pos):
    w = World(19, 8, 2, 96, [pos], [38])
    x = qkv_of(w)
    x[37, :] = math.nan  # q, K and V of the last row
    w.append(x)
    q = q_of(w)
    out = w.attend(q, max_ctx=LONG)
    assert w.status() == 0
    free = (pos + 37) // 16 * 16 - pos  # rows before the lost block
    ref = Cache(w.d_codes.cpu(), w.d_scales.cpu())
    kv = ref.read(0, w.table[w.slots[0]], pos + free)
    for j in range(free):
        want, tol = attention(q[j].cpu().view(w.nq, w.hd), kv, pos + j)
        assert ((out[j].cpu().double().view(w.nq, w.hd) - want).abs() <= tol).all()
    assert out[free:].isnan().all()
    # V alone lost, and K alone
    for kv in (0, 1):
        w.append(qkv_of(w))
        w.d_scales.copy_(w.scales)
        w.d_scales[int(w.table[w.slots[0], 0]), 0, kv, 1, 0] = math.nan
        out = w.attend(q, max_ctx=LONG).view(38, 2, -1)
        assert out[:, 1].isnan().all() and not out[:, 0].isnan().any()


def test_long_runs_report_bad_pages_slots_and_rows():
    def fresh():
        return World(33, 8, 2, 64, [100, 40, 70], [20, 30, 9], unused=(2,))

    for page in (-1, 1 << 30):
        w = fresh()
        w.append(qkv_of(w))
        q = q_of(w)
        good = w.attend(q, max_ctx=LONG)
        assert w.status() == 0
        w.d_table[w.slots[0], 0] = page if page < 0 else w.n_pages
        out = w.attend(q, max_ctx=LONG)
        assert w.status() == DEVICE_ERROR and b"page" in lib().mmc_last_error() and w.status() == 0
        assert torch.equal(out[20:], good[20:]) and not out[:20].isnan().any()
        w.d_table[w.slots[0], :] = -1  # nothing that it could see
        out = w.attend(q, max_ctx=LONG)
        assert w.status() == DEVICE_ERROR and (out[:20] == 0).all() and torch.equal(out[20:], good[20:])
    w = fresh()
    w.d_slots[0] = w.max_seqs
    out = w.attend(q, max_ctx=LONG)
    assert w.status() == DEVICE_ERROR and b"slot" in lib().mmc_last_error()
    assert (out[:20] == 7).all() and not (out[20:50] == 7).any() and (out[50:] == 0).all()
    for pos in (-1, w.max_pages * PAGE - 1, 2 ** 31 - 1):
        w = fresh()
        w.d_pos[w.slots[0]] = pos
        out = w.attend(q, max_ctx=LONG)
        assert w.status() == DEVICE_ERROR and (out[:20] == 7).all() and not (out[20:] == 7).any()
    for start in ([0, 20, 70, 59], [0, -2, 3, 59], [-1, 20, 50, 59], [0, 5, 50, 59], [0, 20, 2 ** 31 - 1, 59]):
        w = fresh()
        w.d_start.copy_(torch.tensor(start, dtype=torch.int32))
        w.attend(q, max_ctx=LONG)
        assert w.status() == DEVICE_ERROR


def test_long_runs_repeat_from_a_graph_and_at_once():
    """The same bits from call to call, from a replayed graph, and from two calls at once with a workspace each."""
    w = World(41, 8, 2, 96, [700, 0, 33], [40, 200, 7])
    w.append(qkv_of(w))
    q = q_of(w)
    first = w.attend(q, max_ctx=LONG)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    bufs = [(torch.empty_like(first), w.workspace(LONG)) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (out, ws) in zip((a, b), bufs):
            w.attend(q, out, ws, C.c_void_p(s.cuda_stream), LONG)
    torch.cuda.synchronize()
    assert w.status() == 0 and torch.equal(bufs[0][0], first) and torch.equal(bufs[1][0], first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=a):
        w.attend(q, *bufs[0], C.c_void_p(a.cuda_stream), LONG)
    # a replay with other lengths: the graph holds none
    w.d_pos[w.slots[0]] = 630
    bufs[0][0].zero_()
    g.replay()
    again = w.attend(q, max_ctx=LONG)
    assert w.status() == 0 and torch.equal(bufs[0][0], again)
    w.pos[0] = 630
    w.check_attention(q, again)


def test_bad_pages_slots_and_rows_are_reported():
    """Device-side refusals: each is reported once, then the word is clear; nothing outside is touched."""
    def fresh():
        return World(31, 8, 2, 64, [100, 40], [2, 3])

    w = fresh()
    w.d_table[w.slots[0], 1] = w.n_pages  # the page of positions 64..127
    before = w.d_codes.clone()
    w.append(qkv_of(w))
    assert w.status() == DEVICE_ERROR and b"page" in lib().mmc_last_error() and w.status() == 0
    w.attend(q_of(w))
    assert w.status() == DEVICE_ERROR and b"page" in lib().mmc_last_error() and w.status() == 0
    other = [p for p in w.table[w.slots[1]].tolist() if p >= 0]
    rest = [p for p in range(w.n_pages) if p not in other]
    assert torch.equal(w.d_codes[rest], before[rest])

    w = fresh()
    w.d_slots[0] = w.max_seqs
    q = w.append(qkv_of(w))
    assert w.status() == DEVICE_ERROR and b"slot" in lib().mmc_last_error()
    out = w.attend(q_of(w))
    assert w.status() == DEVICE_ERROR and (out[:2] == 7).all() and (q[:2] == 7).all() and not (out[2:] == 7).any()

    w = fresh()
    w.d_slots[0] = w.d_slots[1]
    before = w.d_codes.clone()
    w.append(qkv_of(w))
    assert w.status() == DEVICE_ERROR and b"same slot" in lib().mmc_last_error()
    assert torch.equal(w.d_codes, before)

    for pos in (-1, w.max_pages * PAGE - 1, 2 ** 31 - 1):
        w = fresh()
        w.d_pos[w.slots[0]] = pos
        before = w.d_codes.clone()
        w.append(qkv_of(w))
        assert w.status() == DEVICE_ERROR
        out = w.attend(q_of(w))
        assert w.status() == DEVICE_ERROR and (out[:2] == 7).all()

    for start in ([0, 2, 6], [0, -2, 3], [-1, 2, 5], [0, 5, 5], [0, 2, 2 ** 31 - 1]):
        w = fresh()
        w.d_start.copy_(torch.tensor(start, dtype=torch.int32))
        w.append(qkv_of(w))
        w.status()
        w.attend(q_of(w))
        assert w.status() == DEVICE_ERROR

    w = fresh()
    w.max_ctx -= 1
    w.attend(q_of(w), max_ctx=w.max_ctx)
    assert w.status() == DEVICE_ERROR and b"max_ctx" in lib().mmc_last_error()


def test_a_row_range_that_runs_backwards_is_reported_by_append():
    w = World(34, 8, 2, 64, [100, 40, 70], [2, 3, 1])
    w.d_start.copy_(torch.tensor([0, 5, 2, 6], dtype=torch.int32))
    w.max_new = 5
    w.append(qkv_of(w))
    assert w.status() == DEVICE_ERROR and b"row range" in lib().mmc_last_error() and w.status() == 0


def test_small_workspace_and_host_memory_are_refused():
    w = World(1, 8, 2, 64, [3000], [1])
    q, n = q_of(w), w.workspace().numel()
    if n > 16:
        out = torch.empty_like(q)
        assert lib().mmc_op_kv8_attention(w.cache, 0, 1, 1, 1, ptr(w.d_slots), None, 8, ptr(q), w.max_ctx, ptr(out),
                                          ptr(out), n - 1, None) == 1
    host = torch.zeros(1 << 12)
    aligned = (host.data_ptr() + 63) // 64 * 64
    assert lib().mmc_op_kv8_attention(w.cache, 0, 1, 1, 1, ptr(w.d_slots), None, 8, aligned, w.max_ctx, ptr(q), ptr(q),
                                      1 << 30, None) == 1
    assert lib().mmc_op_w4_projection(1, 16, 64, 64, aligned, ptr(q), None, ptr(q), ptr(q), None) == 1


# ------------------------------------------------------------------ 4-bit projections

def w4_case(n, k, batch, group, zeros, seed=0, big=False):
    g = torch.Generator().manual_seed(n * 3 + k + batch + seed)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=g)
    scales = (0.01 * torch.exp(torch.randn(n, k // group, generator=g))).half()
    z = torch.randint(0, 256 if big else 16, (n, k // group), dtype=torch.uint8, generator=g) if zeros else None
    x = (torch.randn(batch, k, generator=g) * torch.exp(torch.randn(k, generator=g))).half()
    return codes, scales, z, x


def w4_run(codes, scales, z, x, group, stream=None, y=None):
    d = [t.cuda() if t is not None else None for t in (codes, scales, z, x)]
    n, b, k = codes.shape[0], x.shape[0], x.shape[1]
    y = torch.full((b + 1, n), 7.0, device="cuda") if y is None else y
    check(lib().mmc_op_w4_projection(b, n, k, group, *(ptr(t) for t in d), ptr(y), stream))
    torch.cuda.synchronize()
    assert (y[b:] == 7).all()
    return y[:b].cpu().double()


def w4_check(codes, scales, z, x, group):
    y = w4_run(codes, scales, z, x, group)
    w = w4_weights(codes, scales, z, group)
    want = x.double() @ w.T
    # products are exact; every value passes at most group / 16 sums of a group, k / group sums over groups and 16 joins,
    # each off by 2^-23 (truncating adders) of what it holds at most: sum |w x|
    k = x.shape[1]
    tol = (group // 16 + 16 + k // group + 32) * 2.0 ** -23 * (x.double().abs() @ w.abs().T) + 1e-30
    assert ((y - want).abs() <= tol).all(), float(((y - want).abs() / tol).max())


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(768, 768), (1152, 768), (17, 128), (1, 128), (2048, 768), (100, 2432), (515, 1408)])
@pytest.mark.parametrize("batch", [1, 3, 8, 9, 24, 64])
def test_w4_projection(n, k, batch, group, zeros):
    if k % group:
        pytest.skip("group does not divide k")
    w4_check(*w4_case(n, k, batch, group, zeros, big=n == 17), group)


@pytest.mark.parametrize("n,k,batch,group,zeros", [(16, 32, 1, 32, True), (5, 96, 2, 32, False), (33, 160, 7, 32, True),
                                                   (300, 16384, 1, 128, False), (64, 8192, 17, 64, True),
                                                   (40, 768, 130, 32, True), (4096, 4096, 33, 128, False),
                                                   (6400, 768, 65, 64, True), (20000, 256, 5, 32, False)])
def test_w4_projection_sizes(n, k, batch, group, zeros):
    w4_check(*w4_case(n, k, batch, group, zeros), group)


@pytest.mark.parametrize("n,k,batch,group,zeros", [
    (6150, 4096, 1, 128, False), (6150, 4096, 5, 64, True), (12300, 4064, 8, 32, True), (16390, 2048, 2, 128, True),
    (32000, 2048, 8, 32, False), (9600, 5120, 3, 64, False)])
def test_w4_projection_of_many_rows_of_weights(n, k, batch, group, zeros):
    """Sizes at which a CTA has several row tiles and as many warps as its registers hold; odd ends of both."""
    w4_check(*w4_case(n, k, batch, group, zeros), group)


def test_w4_projection_repeats_and_special_values():
    """Equal runs give equal bits; an infinite scale or input shows only in its own outputs."""
    codes, scales, z, x = w4_case(200, 512, 5, 64, True)
    a = w4_run(codes, scales, z, x, 64)
    for _ in range(3):
        assert torch.equal(a, w4_run(codes, scales, z, x, 64))
    scales[7, 3] = math.nan
    x[2, 100] = math.inf
    b = w4_run(codes, scales, z, x, 64)
    assert b[:, 7].isnan().all() and not torch.isfinite(b[2]).any()
    keep = torch.ones_like(a, dtype=torch.bool)
    keep[:, 7] = False
    keep[2] = False
    assert torch.equal(a[keep], b[keep])


# ------------------------------------------------------------------ a run of them together

def test_quantised_block_runs_together():
    """The attention block of a small model with 4-bit weights and the 8-bit cache: a prompt pass and single steps of
    ragged sequences. Each operator's output is checked against its 64-bit form on the inputs it found; the steps are
    then repeated from the same state as one captured graph, on another stream, with equal bits."""
    hidden, nq, nkv, hd, group = 256, 8, 2, 64, 64
    qdim, odim = (nq + 2 * nkv) * hd, nq * hd
    pos, new = [0, 0, 0], [37, 5, 64]
    w = World(77, nq, nkv, hd, [80, 80, 80], [1, 1, 1])  # pages for 80 positions and more
    qn, kn = [t.cuda() for t in norms_of(w)]
    W = {}
    for name, n, k in (("qkv", qdim, hidden), ("o", hidden, odim)):
        c, s, z, _ = w4_case(n, k, 1, group, True)
        W[name] = (c, s * 0.3, z, [t.cuda() for t in (c, s * 0.3, z)])

    def project(name, x, y, stream=None):
        c, s, z, d = W[name]
        check(lib().mmc_op_w4_projection(x.shape[0], c.shape[0], x.shape[1], group, *(ptr(t) for t in d), ptr(x), ptr(y),
                                         stream))

    def check_project(name, x, y):
        c, s, z, _ = W[name]
        wt = w4_weights(c, s, z, group)
        xs = x.cpu().double()
        tol = (group // 16 + 16 + x.shape[1] // group + 32) * 2.0 ** -23 * (xs.abs() @ wt.abs().T) + 1e-30
        assert ((y.cpu().double() - xs @ wt.T).abs() <= tol).all()

    def step(x, checked):
        """x [rows][hidden] fp16 -> the block's output, every stage checked."""
        y = torch.empty(w.rows, qdim, device="cuda")
        o = torch.empty(w.rows, hidden, device="cuda")
        project("qkv", x, y)
        w.codes, w.scales = w.d_codes.cpu(), w.d_scales.cpu()
        q = w.append(y, qn, kn)
        att = w.attend(q)
        project("o", att, o)
        assert w.status() == 0
        if checked:
            check_project("qkv", x, y)
            w.check_append(y, qn.cpu(), kn.cpu(), q)
            w.check_attention(q, att)
            check_project("o", att, o)
        return o

    def batch(pos, new):
        w.pos, w.new = list(pos), list(new)
        w.start = [0]
        for n in new:
            w.start.append(w.start[-1] + n)
        w.rows, w.max_new = w.start[-1], max(new)
        w.d_start.copy_(torch.tensor(w.start, dtype=torch.int32))
        for i, s in enumerate(w.slots):
            w.d_pos[s] = pos[i]

    batch(pos, new)
    x = torch.randn(w.rows, hidden, generator=w.g).half().cuda()
    step(x, True)
    pos = [p + n for p, n in zip(pos, new)]
    saved, steps = None, []
    for i in range(6):
        batch(pos, [1, 1, 1])
        if i == 0:
            saved = w.d_codes.clone(), w.d_scales.clone(), w.d_pos.clone()
        x = torch.randn(3, hidden, generator=w.g).half().cuda()
        steps.append((x, step(x, True)))
        pos = [p + 1 for p in pos]
    # the same steps as replays of one graph
    w.d_codes.copy_(saved[0])
    w.d_scales.copy_(saved[1])
    w.d_pos.copy_(saved[2])
    xs = torch.empty(3, hidden, dtype=torch.float16, device="cuda")
    y = torch.empty(3, qdim, device="cuda")
    q, att = (torch.empty(3, odim, dtype=torch.float16, device="cuda") for _ in range(2))
    o = torch.empty(3, hidden, device="cuda")
    ws = w.workspace()
    idx = torch.tensor(w.slots, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        s = torch.cuda.current_stream().cuda_stream
        project("qkv", xs, y, s)
        w.append(y, qn, kn, q, s)
        w.attend(q, att, ws, s)
        project("o", att, o, s)
        w.d_pos[idx] += 1
    torch.cuda.synchronize()
    for x, want in steps:
        xs.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)
    assert w.status() == 0


def test_two_streams_with_a_workspace_each():
    """Calls side by side on two streams, each with its own workspace and outputs, equal the calls alone."""
    ws = [World(s, 8, 2, 96, [1500 + s, 300], [1, 1]) for s in (1, 2)]
    qs = [q_of(w) for w in ws]
    for w in ws:
        w.append(qkv_of(w))
    alone = [w.attend(q) for w, q in zip(ws, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ws]
    space = [w.workspace() for w in ws]
    outs = [torch.full_like(a, 7.0) for a in alone]
    torch.cuda.synchronize()
    for _ in range(20):
        for w, q, s, sp, o in zip(ws, qs, streams, space, outs):
            w.attend(q, o, sp, s.cuda_stream)
    torch.cuda.synchronize()
    for a, o in zip(alone, outs):
        assert torch.equal(a, o)


@pytest.mark.parametrize("new,max_ctx", [([1, 1], None), ([5, 1], None), ([40, 3], LONG)])
def test_cache_of_more_than_4_gib(new, max_ctx):
    """Pages behind the first 2^32 bytes of the codes: the same bits as from a small cache."""
    w = World(50, 16, 8, 128, [200, 70], new, layers=4, layer=3)
    x, q = qkv_of(w), q_of(w)
    w.append(x)
    out = w.attend(q, max_ctx=max_ctx)
    page = w.codes[0].numel()
    n = (1 << 32) // page + 2 * w.n_pages
    big = World(50, 16, 8, 128, [200, 70], new, layers=4, layer=3)
    first = n - big.n_pages
    codes = torch.empty((n, *big.codes.shape[1:]), dtype=torch.uint8, device="cuda")
    scales = torch.empty((n, *big.scales.shape[1:]), device="cuda")
    codes[first:], scales[first:] = big.codes.cuda(), big.scales.cuda()
    big.d_table[big.d_table >= 0] += first
    big.cache.n_pages, big.cache.d_codes, big.cache.d_scales = n, ptr(codes), ptr(scales)
    big.append(x)
    assert torch.equal(big.attend(q, max_ctx=max_ctx), out)
    assert w.status() == 0 and big.status() == 0
    assert torch.equal(codes[first:], w.d_codes) and torch.equal(scales[first:], w.d_scales)


@pytest.mark.parametrize("batch", [1, 9])
def test_w4_projection_of_more_than_4_gib(batch):
    """Codes behind the first 2^32 bytes, with products and sums of whole numbers: exact."""
    n, k, group = (1 << 26) + 40, 128, 64
    g = torch.Generator(device="cuda").manual_seed(60)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.exp2(torch.randint(-2, 2, (n, k // group), device="cuda", generator=g).float()).half()
    x = torch.randint(-4, 5, (batch, k), device="cuda", generator=g).half()
    y = torch.empty(batch, n, device="cuda")
    check(lib().mmc_op_w4_projection(batch, n, k, group, ptr(codes), ptr(scales), None, ptr(x), ptr(y), None))
    for rows in (slice(0, 100), slice(n // 2, n // 2 + 100), slice(n - 300, n)):
        want = x.double().cpu() @ w4_weights(codes[rows].cpu(), scales[rows].cpu(), None, group).T
        assert torch.equal(y[:, rows].double().cpu(), want)


# ------------------------------------------------------------------ a large max_ctx and short sequences

@pytest.mark.parametrize("max_ctx", [1500, 4000, LONG])
@pytest.mark.parametrize("rows", ["steps", "several", "unused"])
def test_next_node_of_a_graph_finds_the_rows(rows, max_ctx):
    """A captured call whose max_ctx is the capacity: several parts by its plan, while every sequence has one (or none
    has rows). The graph's next node reads the rows at once, in each of many replays over a cleared buffer."""
    new = {"steps": [1] * 24, "several": [3, 5, 1] * 8, "unused": [11] * 24}[rows]
    pos = [(i * 37) % 180 for i in range(24)]
    w = World(90, 8, 2, 96, pos, new, unused=range(24) if rows == "unused" else ())
    w.append(qkv_of(w))
    q = q_of(w)
    alone = w.attend(q)
    w.check_attention(q, alone)
    ws, out, seen = w.workspace(max_ctx), torch.empty_like(alone), torch.empty_like(alone)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        for _ in range(4):
            out.fill_(7.0)
            w.attend(q, out, ws, st.cuda_stream, max_ctx)
            seen.copy_(out)
    g.replay()
    torch.cuda.synchronize()
    w.check_attention(q, seen)
    first = seen.clone()
    for _ in range(50):
        seen.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(seen, first)
    assert w.status() == 0


# ------------------------------------------------------------------ V blocks of zeros and of very different sizes

# pages of a sequence whose V blocks are zeros (scale 2^-126, as the append stores them) or of the scale 2^-120, among
# ordinary positive ones
QUIET_PAGES = {"first": [0], "first two": [0, 1], "middle": [5], "two running": [3, 4], "four running": [4, 5, 6, 7],
               "all but one": [p for p in range(17) if p != 2], "every other": list(range(0, 17, 2))}


def quieten(w, pages, what, head):
    """V of kv head `head` in those pages (of each sequence that has them): zeros, 2^-120, or the two in turn."""
    w.d_codes[:, :, 1] &= 0x7f
    for s in w.slots:
        for n, j in enumerate(j for j in pages if j < w.max_pages and int(w.table[s, j]) >= 0):
            at = int(w.table[s, j]), w.layer, 1, head
            zero = what == "zeros" or (what == "both" and n % 2 == 0)
            w.d_scales[at] = 2.0 ** (-126 if zero else -120)
            if zero:
                w.d_codes[at] = 0


def quiet_case(hd, new, pages, what, max_ctx=None):
    w = World(hd + 3, 8, 2, hd, [1000, 64, 333], new)
    w.append(qkv_of(w))
    quieten(w, QUIET_PAGES[pages], what, 0)
    q = q_of(w)
    out = w.attend(q, max_ctx=max_ctx)
    assert w.status() == 0
    w.check_attention(q, out)


@pytest.mark.parametrize("what", ["zeros", "tiny", "both"])
@pytest.mark.parametrize("pages", QUIET_PAGES)
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 2, 5]])
@pytest.mark.parametrize("hd", [16, 32, 64, 96, 128])
def test_zero_and_tiny_values_among_ordinary_ones(hd, new, pages, what):
    quiet_case(hd, new, pages, what)


@pytest.mark.parametrize("gap", [21, 60, 90, 100, 126, 127, 135])
@pytest.mark.parametrize("hd", [32, 96, 128])
def test_values_that_grow_or_fall_block_by_block(hd, gap):
    """V's scales up and down by 2^gap between 2^-126 and 2^9, a block at a time and a page at a time; outputs go by the
    largest blocks, and those that see none of them by the small ones."""
    for step in (1, 4):
        w = World(hd + gap, 8, 2, hd, [900, 63, 200], [2, 1, 3], size=2.0 ** 7)
        w.append(qkv_of(w, 16.0))
        e = [9, 9 - gap, 9, 9, 9 - gap, 9 - gap, 9 - gap // 2, 9]
        for s in w.slots:
            for j, p in enumerate(int(p) for p in w.table[s] if p >= 0):
                for b in range(4):
                    w.d_scales[p, 0, 1, :, b] = 2.0 ** max(-126, e[(4 * j + b) // step % 8] - 7)
        q = q_of(w)
        out = w.attend(q)
        assert w.status() == 0
        w.check_attention(q, out)


@pytest.mark.parametrize("what", ["zeros", "tiny", "both"])
@pytest.mark.parametrize("pages", QUIET_PAGES)
@pytest.mark.parametrize("hd", [16, 32, 64, 96, 128])
def test_long_runs_zero_and_tiny_values_among_ordinary_ones(hd, pages, what):
    quiet_case(hd, [40, 30, 50], pages, what, LONG)


@pytest.mark.parametrize("scales", [(0, -60, -120), (0, -63, -64, -65, -84, -85, -86, -126), (0, -40, -80, -119, -20),
                                    (-126, -100, -60, -20, 0, -85, -126)])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_long_runs_falling_and_growing_values(hd, scales):
    """V's scales page by page, and block by block: 1 to 2^-126 of the largest one."""
    for step in (1, 4):
        w = World(hd + len(scales), 8, 2, hd, [1000, 63, 200], [40, 33, 36])
        w.append(qkv_of(w))
        w.d_codes[:, :, 1] &= 0x7f
        for s in w.slots:
            for j, p in enumerate(int(p) for p in w.table[s] if p >= 0):
                for b in range(4):
                    w.d_scales[p, 0, 1, :, b] = 2.0 ** max(-126, scales[(4 * j + b) // step % len(scales)] - 4)
        q = q_of(w)
        out = w.attend(q, max_ctx=LONG)
        assert w.status() == 0
        w.check_attention(q, out)


@pytest.mark.parametrize("scale", [-1.0, 0.0, -0.0, math.inf, -math.inf, math.nan, -2.0 ** 100])
@pytest.mark.parametrize("new,max_ctx", [([1, 1, 1], None), ([3, 2, 5], None), ([40, 7, 33], LONG)])
def test_blocks_without_positions_hold_anything(new, max_ctx, scale):
    """Codes and scales have no initial values: blocks that no position has been written to hold any scale and any code."""
    for hd in (64, 96):
        w = World(60 + hd, 8, 2, hd, [129, 70, 300], new)
        kept = torch.zeros_like(w.scales, dtype=torch.bool)
        for i, s in enumerate(w.slots):
            for b in range(-(-w.pos[i] // 16)):
                kept[int(w.table[s, b // 4]), ..., b % 4] = True
        w.scales[~kept] = scale
        w.d_scales.copy_(w.scales)
        x = qkv_of(w)
        qn, kn = norms_of(w)
        qa = w.append(x, qn.cuda(), kn.cuda())
        assert w.status() == 0
        w.check_append(x, qn, kn, qa)
        q = q_of(w)
        out = w.attend(q, max_ctx=max_ctx)
        assert w.status() == 0
        w.check_attention(q, out)


# ------------------------------------------------------------------ small weights

def small_weights(w, log2p, hidden):
    """All of sequence 0's scores 0 but for those of the first positions of two pages' blocks, which are so far above them
    that the weights are 2^log2p of theirs; values 1 to 4 eighths. `hidden`: pages whose V is 64 times larger and whose
    weights are 0."""
    g = w.g
    w.d_codes[:, :, 0] = 0
    w.d_codes[:, :, 1] = torch.randint(0x38, 0x48, w.d_codes[:, :, 1].shape, dtype=torch.uint8, generator=g).cuda()
    w.d_scales[:, :, 0] = 1.0
    w.d_scales[:, :, 1] = 0.125
    row = w.table[w.slots[0]]
    for j in hidden:
        w.d_codes[int(row[j]), :, 0] = 0xfe  # -448
        w.d_scales[int(row[j]), :, 1] = 8.0
    for j in (0, (2 * w.max_pages) // 3 // 4 * 4 + 2):  # in each warp's share of each of two parts
        w.d_codes[int(row[j]), :, 0, :, ::16] = 0x38  # 1
    a = -log2p * math.log(2.0) / math.sqrt(w.hd)
    return torch.full((w.rows, w.nq * w.hd), a, dtype=torch.float16, device="cuda")


@pytest.mark.parametrize("hd,pos,new,log2p,hide", [(64, 24000, 1, -14.914, True), (96, 24000, 4, -14.914, True),
                                                   (128, 24000, 1, -13.914, True), (32, 300000, 1, -19.64, False)])
def test_many_small_weights_keep_their_bits(hd, pos, new, log2p, hide):
    """Positions that weigh 2^-15 or 2^-19 of the largest each, thousands of them a warp and part (a padded batch is
    split into few parts): rounded to 2^-11 of each weight as larger ones are, so that an output is within 2^-11 of its
    size and its own half step. fp32's part: 2^-14, and chains of pos / 32 additions of weights (2^-24 each) and of pos / 64
    of products (2^-23, as they are truncated)."""
    n = 2000
    w = World(81, 4, 1, hd, [pos] + [0] * (n - 1), [new] * n, unused=range(1, n))
    w.append(qkv_of(w))
    pages = -(-(pos + new) // PAGE)
    q = small_weights(w, log2p, range(1, pages - 1, 4) if hide else ())
    out = w.attend(q)[:new].cpu().double().view(new, 4, hd)
    assert w.status() == 0
    kv = Cache(w.d_codes.cpu(), w.d_scales.cpu()).read(0, w.table[w.slots[0]], pos + new)
    for j in range(new):
        want, _ = attention(q[j].cpu().view(4, hd), kv, pos + j)
        off = (out[j] - want).abs() / want.abs()
        assert (off <= 2.0 ** -10 + 2.0 ** -14 + pos * 2.0 ** -28).all()


def test_rows_of_no_sequence_have_no_effect():
    """Rows of the buffers behind the last sequence, between none, and of unused sequences hold NaN: nothing shows it."""
    for new, max_ctx in (([1, 1, 1, 1], None), ([3, 2, 1, 4], None), ([40, 7, 33, 20], LONG)):
        w = World(15, 8, 2, 64, [70, 10, 33, 5], new, spare_rows=9, unused=(1, 3))
        x, q = qkv_of(w), q_of(w)
        for i in (1, 3):
            x[w.start[i]:w.start[i + 1]] = q[w.start[i]:w.start[i + 1]] = math.nan
        x[w.start[-1]:] = q[w.start[-1]:] = math.nan
        got = w.append(x, start=ptr(w.d_start))
        assert w.status() == 0 and (got[w.start[-1]:] == 7).all()
        w.check_append(x, None, None, got)
        out = w.attend(q, max_ctx=max_ctx)
        assert w.status() == 0
        w.check_attention(q, out)


@pytest.mark.parametrize("hd", [64, 96])
def test_proposals_that_are_given_up(hd):
    """Rows appended, rejected by lowering the position, and others appended in their place: each call equals the
    64-bit form on the cache that it found (a block keeps the scale that rejected rows have raised, the older values
    stay). A block that is begun anew has a scale of its own, even behind a NaN."""
    pos = [30, 64, 13]
    w = World(71 + hd, 8, 2, hd, pos, [5, 5, 5])
    for size, bad in ((50.0, None), (1.0, None), (1.0, math.nan), (2.0, None)):
        x = qkv_of(w, size)
        if bad is not None:
            x[9, :] = bad  # the last row of the sequence at position 64, whose block begins with the call
        w.codes, w.scales = w.d_codes.cpu(), w.d_scales.cpu()
        qa = w.append(x)
        assert w.status() == 0
        if bad is None:
            w.check_append(x, None, None, qa)
            q = q_of(w)
            out = w.attend(q)
            assert w.status() == 0
            w.check_attention(q, out)
        # (the device's positions were not advanced: the next call's rows take the place of these)


# ------------------------------------------------------------------ borders, first calls, far sizes

@pytest.mark.parametrize("amax", [448.0, 448.00003, 449.0, 3.4e38, 1.75 * 2.0 ** -126, 1e-40, 1e-45, 0.0])
def test_values_at_scale_borders_are_all_numbers(amax):
    """Every V code that an append writes, and every older one of its blocks, is the 64-bit form's; none becomes a NaN."""
    w = World(3, 2, 2, 32, [3, 16], [2, 1])
    x = qkv_of(w, 0.1 * min(amax, 1e37))
    x[:, -w.nkv * w.hd:].clamp_(-amax, amax)
    x[0, -1] = amax
    x[2, -w.hd - 5] = -amax
    w.append(x)
    assert w.status() == 0
    ref = Cache(w.codes, w.scales)
    v = x.cpu().view(w.rows, w.nq + 2 * w.nkv, w.hd)[:, -w.nkv:].double()
    got = e4m3_table()[w.d_codes.cpu().long()]
    for i in range(w.seqs):
        vi = v[w.start[i]:w.start[i + 1]].transpose(0, 1)
        ref.append(0, w.table[w.slots[i]], w.pos[i], torch.stack([vi, vi]))
        for p in range(w.pos[i] + w.new[i]):
            page = int(w.table[w.slots[i], p // PAGE])
            assert torch.equal(got[page, 0, 1, :, p % PAGE], ref.codes[page, 0, 1, :, p % PAGE])


FIRST_CALL = """
import ctypes as C, sys, torch
sys.path[:0] = [{tests!r}, {root!r}]
import test_gpu_lowbit as T
kind = {kind!r}
st = torch.cuda.Stream()
if kind == "projection":
    codes, scales, z, x = [t.cuda() for t in T.w4_case(300, 512, {n}, 64, True)]
    y = torch.zeros({n}, 300, device="cuda")
    def call(s):
        T.check(T.lib().mmc_op_w4_projection({n}, 300, 512, 64, *(T.ptr(t) for t in (codes, scales, z, x, y)), s))
    result = lambda: y
else:
    w = T.World(3, 8, 2, 64, [70 + {n}, 200 + {n}, 33 + {n}], [{n}] * 3)
    w.d_pos -= {n}  # the rows' own positions hold values
    x, q = T.qkv_of(w), T.q_of(w)
    out = torch.full_like(q, 7.0)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    if kind == "append":
        call = lambda s: w.append(x, None, None, out, s)
        result = lambda: torch.cat([out.view(torch.uint8).flatten(), w.d_codes.flatten()])
    else:
        call = lambda s: w.attend(q, out, ws, s, {ctx})
        result = lambda: out.view(torch.uint8)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=st):
    call(st.cuda_stream)
g.replay()
torch.cuda.synchronize()
captured = result().clone()
call(None)
torch.cuda.synchronize()
assert torch.equal(captured, result()) and not (captured == 7).all() and bool(captured.any())
print("equal")
"""


@pytest.mark.parametrize("kind,n,ctx", [("projection", 1, 0), ("projection", 20, 0), ("append", 1, 0), ("append", 12, 0),
                                        ("attention", 1, 300), ("attention", 12, LONG)])
def test_the_first_call_of_a_process_is_captured(kind, n, ctx):
    """Nothing has been set up by an eager call before."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = FIRST_CALL.format(tests=here, root=os.path.dirname(here), kind=kind, n=n, ctx=ctx)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("new,max_ctx", [([1, 1], None), ([3, 2], None), ([3, 2], LONG)])
@pytest.mark.parametrize("nq,nkv,hd", [(160, 1, 16), (258, 2, 32), (131, 1, 64), (300, 3, 96)])
def test_groups_of_more_than_a_tile_of_heads(nq, nkv, hd, new, max_ctx):
    w = World(nq + hd, nq, nkv, hd, [130, 61], new)
    x = qkv_of(w)
    qa = w.append(x)
    assert w.status() == 0
    w.check_append(x, None, None, qa)
    q = q_of(w)
    out = w.attend(q, max_ctx=max_ctx)
    assert w.status() == 0
    w.check_attention(q, out)


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 2, 5], [40, 7, 33]])
def test_the_largest_max_ctx(new):
    """2^31 - 1, whatever the sequences hold: the same rows as with a close bound but for the parts' rounding."""
    w = World(70, 8, 2, 96, [700, 70, 1000], new)
    w.append(qkv_of(w))
    q = q_of(w)
    out = w.attend(q, max_ctx=2 ** 31 - 1)
    assert w.status() == 0
    w.check_attention(q, out)


def test_more_sequences_than_threads_and_one_slot_twice_far_apart():
    n = 700
    g = torch.Generator().manual_seed(72)
    pos = torch.randint(0, 100, (n,), generator=g).tolist()
    w = World(73, 4, 2, 32, pos, [1] * n, unused=(3, 600))
    x = qkv_of(w)
    qa = w.append(x)
    assert w.status() == 0
    w.check_append(x, None, None, qa)
    q = q_of(w)
    out = w.attend(q)
    assert w.status() == 0
    w.check_attention(q, out)
    w.d_slots[690] = w.d_slots[12]
    before = w.d_codes.clone()
    qa = w.append(qkv_of(w))
    assert w.status() == DEVICE_ERROR and b"same slot" in lib().mmc_last_error() and w.status() == 0
    touched = [int(w.table[w.slots[i], pos[i] // PAGE]) for i in range(n) if i not in (3, 600, 12, 690)]
    rest = [p for p in range(w.n_pages) if p not in set(touched)]
    assert torch.equal(w.d_codes[rest], before[rest])
    assert (qa[[12, 690]] == 7).all() and not (qa[[11, 691]] == 7).any()




@pytest.mark.parametrize("n,k,batch,group,zeros", [
    (48, 65536, 1, 128, True), (48, 65536, 8, 32, False), (33, 40960, 20, 64, True), (5, 32, 64, 32, True),
    (16 * 148 * 16 + 5, 64, 8, 64, False), (148 * 16 * 3 + 1, 2080, 4, 32, True), (7, 2048, 300, 128, False)])
def test_w4_projection_far_sizes(n, k, batch, group, zeros):
    w4_check(*w4_case(n, k, batch, group, zeros), group)


@pytest.mark.parametrize("batch", [1, 8, 24])
def test_w4_projection_from_odd_places(batch):
    """Scales and zero points at any address of their type, as views of larger arrays have."""
    for n, k, group in ((70, 1024, 32), (70, 2080, 32), (200, 2304, 64)):
        codes, scales, z, x = w4_case(n, k, batch, group, True)
        want = w4_run(codes, scales, z, x, group)
        sc = torch.empty(scales.numel() + 8, dtype=torch.float16, device="cuda")
        zz = torch.empty(z.numel() + 16, dtype=torch.uint8, device="cuda")
        d_codes, d_x = codes.cuda(), x.cuda()
        for o in (1, 2, 3, 4, 7):
            sc[o:o + scales.numel()] = scales.cuda().flatten()
            zz[o:o + z.numel()] = z.cuda().flatten()
            y = torch.empty(batch, n, device="cuda")
            check(lib().mmc_op_w4_projection(batch, n, k, group, ptr(d_codes), ptr(sc) + 2 * o, ptr(zz) + o, ptr(d_x),
                                             ptr(y), None))
            assert torch.equal(y.cpu().double(), want)
