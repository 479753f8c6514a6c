"""The paged KV cache: appending with the rotation on the way, attention over the pages, both and sampling as they are used together."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from bpd_substrate_b200 import capi

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
PAIRS = [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Cache:
    """Sequences' pages in random order in a pool whose unused places hold NaN; K and V may lie in one block (page_stride)."""

    def __init__(self, H, G, D, act, kv, page, held, new, seed=0, ragged=None, joint=False, shared=(), spare_entries=1):
        g = torch.Generator().manual_seed(seed)
        self.H, self.G, self.D, self.act, self.kv, self.page, self.held, self.new = H, G, D, act, kv, page, list(held), list(new)
        self.ragged = max(new, default=1) != 1 or min(new, default=1) != 1 if ragged is None else ragged
        need = [-(-(h + n) // page) for h, n in zip(held, new)]
        self.max_pages = max(need, default=0) + spare_entries
        self.n_pages = sum(need) + 3
        order = torch.randperm(self.n_pages, generator=g).to(torch.int32)
        self.table = torch.full((max(1, len(held)), self.max_pages), 10 ** 6, dtype=torch.int32)          # entries that nobody may follow
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        for first, last, pages in shared:                    # sequences first .. last - 1 begin with the first one's pages
            for b in range(first + 1, last):
                self.table[b, :pages] = self.table[first, :pages]
        stride = G * page * D
        self.stride = 2 * stride + 16 if joint else 0
        t = TYPES[kv][0]
        if joint:
            self.pool = torch.full((self.n_pages, self.stride), float("nan"), dtype=t)
            self.k = self.pool[:, :stride].view(self.n_pages, G, page, D)
            self.v = self.pool[:, stride:2 * stride].view(self.n_pages, G, page, D)
        else:
            self.pool = torch.full((2, self.n_pages, G, page, D), float("nan"), dtype=t)
            self.k, self.v = self.pool[0], self.pool[1]
        self.start = [0]
        for n in new:
            self.start.append(self.start[-1] + n)
        self.tokens = self.start[-1]
        self.gen = g

    def fill(self, everything=True, scale=1.0):
        """Random keys and values at the places that sequences hold; with the new tokens' too if `everything`."""
        for b, (h, n) in enumerate(zip(self.held, self.new)):
            p = torch.arange(h + (n if everything else 0))
            if p.numel():
                rows = self.table[b].long()[p // self.page]
                for x in (self.k, self.v):
                    x[rows, :, p % self.page] = (torch.randn(p.numel(), self.G, self.D, generator=self.gen) * scale).to(x.dtype)

    def upload(self):
        self.d_pool, self.d_table, self.d_len, self.d_start = self.pool.cuda(), self.table.cuda(), i32(self.held or [0]), i32(self.start)
        size = self.pool.element_size()
        k = self.d_pool.data_ptr()
        self.desc = capi.PagedKv(self.H, self.G, self.D, TYPES[self.act][1], TYPES[self.kv][1], self.page, self.n_pages, len(self.held), self.max_pages, self.stride, k,
                                 k + size * (self.G * self.page * self.D if self.stride else self.pool[0].numel()), self.d_table.data_ptr(), self.d_len.data_ptr(),
                                 self.d_start.data_ptr() if self.ragged else None)
        torch.cuda.synchronize()
        return C.byref(self.desc)

    def read(self):
        """(k, v) as they are now."""
        pool = self.d_pool.cpu()
        if not self.stride:
            return pool[0], pool[1]
        n = self.G * self.page * self.D
        return pool[:, :n].view(self.k.shape), pool[:, n:2 * n].view(self.v.shape)


def done(lib, status):
    assert status == 0
    torch.cuda.synchronize()
    assert lib.bpdq_last_status() == 0


# ---- append

def turned(x, pos, rot, neighbours, freq):
    """x [T, heads, D] float64."""
    a = pos[:, None].double() * freq.double()
    c, s = a.cos()[:, None], a.sin()[:, None]
    y = x.clone()
    i = torch.arange(rot // 2)
    p, q = (2 * i, 2 * i + 1) if neighbours else (i, i + rot // 2)
    y[..., p], y[..., q] = x[..., p] * c - x[..., q] * s, x[..., p] * s + x[..., q] * c
    return y


def append_case(lib, H, G, D, act, kv, page, held, new, rot, neighbours, seed=0, ragged=None, joint=False, in_place=True, pad=0, queries=True, slack=0, base=500000.0):
    c = Cache(H, G, D, act, kv, page, held, new, seed, ragged, joint)
    c.fill(everything=False)
    T, ld = c.tokens + pad, (H + 2 * G) * D + slack
    x = torch.randn(T, ld, generator=c.gen).to(TYPES[act][0])
    freq = (base ** (-torch.arange(max(1, rot // 2)).double() / max(1, rot // 2))).float()
    d, dfreq, out = x.cuda(), freq.cuda(), torch.full((T, H * D), 9.0, dtype=x.dtype, device="cuda")
    desc, size = c.upload(), x.element_size()
    before_k, before_v = c.read()
    q = d.data_ptr() if queries else None
    q_out, ld_out = (None, 0) if not queries else ((d.data_ptr(), ld) if in_place else (out.data_ptr(), H * D))
    done(lib, lib.bpd_paged_append_cuda(desc, q, ld, q_out, ld_out, d.data_ptr() + H * D * size, ld, d.data_ptr() + (H + G) * D * size, ld, T, rot, neighbours,
                                        dfreq.data_ptr() if rot else None, None))
    pos = torch.cat([h + torch.arange(n) for h, n in zip(held, new)] or [torch.zeros(0)]).long()
    heads = x[:c.tokens, :(H + 2 * G) * D].double().view(c.tokens, H + 2 * G, D)
    want = heads.clone()
    want[:, :H + G] = turned(heads[:, :H + G], pos, rot, neighbours, freq[:rot // 2])
    # sine and cosine to 2 units, the half turn's rounding (2^-24 of at most 1, times pi), two products and a sum
    length = heads[:, :H + G].abs().amax() * 2

    def tolerance(kind, w):
        return HALF_STEP[kind] * w.abs() + (8 * 2.0 ** -24 * length if rot else 0) + (2.0 ** -25 if kind == "f16" else 0)

    if queries:
        got = (d.cpu()[:, :H * D] if in_place else out.cpu()).double()
        q_want = want[:, :H].reshape(c.tokens, -1)
        assert ((got[:c.tokens] - q_want).abs() <= tolerance(act, q_want)).all()
        rest = x[c.tokens:, :H * D].double() if in_place else torch.full_like(got[c.tokens:], 9.0)
        assert torch.equal(got[c.tokens:], rest)                # rows behind the last sequence
    k, v = c.read()
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(new)] or [torch.zeros(0)]).long()
    rows, slot = c.table.long()[seq, pos // page], pos % page
    assert ((k[rows, :, slot].double() - want[:, H:H + G]).abs() <= tolerance(kv, want[:, H:H + G])).all()
    assert torch.equal(v[rows, :, slot], heads[:, H + G:].to(v.dtype))
    before_k[rows, :, slot], before_v[rows, :, slot] = k[rows, :, slot], v[rows, :, slot]
    assert torch.equal(k.view(torch.int16), before_k.view(torch.int16)) and torch.equal(v.view(torch.int16), before_v.view(torch.int16))      # nothing else was touched


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("neighbours", [0, 1])
@pytest.mark.parametrize("H,G,D,rot,page", [(4, 2, 64, 64, 16), (3, 3, 128, 64, 8), (8, 1, 96, 96, 32), (14, 2, 64, 32, 128), (2, 1, 80, 20, 16), (6, 2, 8, 2, 256), (5, 5, 40, 0, 64)])
def test_append(lib, act, kv, neighbours, H, G, D, rot, page):
    append_case(lib, H, G, D, act, kv, page, [0, 3, page, 2 * page - 1], [1, 1, 1, 1], rot, neighbours, seed=rot)
    append_case(lib, H, G, D, act, kv, page, [0, 3, page - 1, 77], [page + 3, 1, 0, 2], rot, neighbours, seed=D, pad=3)


@pytest.mark.parametrize("act,kv", PAIRS)
def test_append_forms(lib, act, kv):
    """Queries elsewhere, none, rows with odd strides, pools in one block, one token per sequence behind bounds, spare rows."""
    for i, form in enumerate([dict(in_place=False), dict(queries=False), dict(slack=1), dict(slack=4), dict(joint=True), dict(ragged=True), dict(pad=5), dict(ragged=True, pad=2, in_place=False)]):
        append_case(lib, 6, 2, 64, act, kv, 16, [5, 40, 100], [1, 1, 1], 64, i & 1, seed=i, **form)


def test_append_far_positions(lib):
    """Positions of a million turn as exactly as the first ones."""
    append_case(lib, 2, 1, 64, "f32", "f16", 256, [1000003, 524287], [2, 1], 64, 1)
    append_case(lib, 2, 1, 64, "f32", "f16", 256, [1000003, 524287], [2, 1], 64, 0, base=3.0)


def test_append_many_sequences(lib):
    rng = np.random.default_rng(1)
    new = rng.integers(0, 4, 700).tolist()
    append_case(lib, 2, 1, 32, "bf16", "bf16", 8, rng.integers(0, 30, 700).tolist(), new, 32, 0, pad=1)
    append_case(lib, 2, 1, 32, "bf16", "bf16", 8, rng.integers(0, 30, 2048).tolist(), [1] * 2048, 32, 1)


def test_append_skips_what_makes_no_sense(lib):
    """Bad lengths, bounds and pages: the rows and pages concerned stay, the rest is right, and the status says so."""
    c = Cache(2, 1, 64, "bf16", "bf16", 8, [5, 9, 3, 4, 6], [2, 2, 2, 2, 2], 3)
    c.fill(everything=False)
    c.table[3, 0] = c.n_pages                      # of sequence 3: positions 4 and 5
    c.table[4, 0] = -1
    c.held = [5, -1, 8 * c.max_pages - 1, 4, 6]
    desc = c.upload()
    before_k, _ = c.read()
    x = torch.randn(10, 4 * 64, generator=c.gen).bfloat16()
    d = x.cuda()
    assert lib.bpd_paged_append_cuda(desc, d.data_ptr(), 256, d.data_ptr(), 256, d.data_ptr() + 256, 256, d.data_ptr() + 384, 256, 10, 0, 0, None, None) == 0
    torch.cuda.synchronize()
    assert lib.bpdq_last_status() == -4
    lib.bpdq_clear_status()
    k, _ = c.read()
    page, slot = c.table[0, 0].long(), [5, 6]
    assert torch.equal(k[page, 0, slot], x[:2, 128:192])
    before_k[page, 0, slot] = k[page, 0, slot]
    assert torch.equal(k.view(torch.int16), before_k.view(torch.int16))
    c.d_start.copy_(i32([0, 2, 11, 4, 3, 9 ** 9]))
    torch.cuda.synchronize()
    assert lib.bpd_paged_append_cuda(desc, None, 0, None, 0, d.data_ptr() + 256, 256, d.data_ptr() + 384, 256, 10, 0, 0, None, None) == 0
    torch.cuda.synchronize()
    assert lib.bpdq_last_status() == -4
    lib.bpdq_clear_status()


# ---- attention

def attention_oracle(c, q, scale, cap, missing=()):
    """(o, bound) [T, H, D] in 64 bits: bound = sum of w |v| (what errors of weights are relative to) and the rows' largest sum of |q k|."""
    T, share = c.tokens, c.H // c.G
    out, size, top = (torch.zeros(T, c.H, c.D, dtype=torch.float64, device="cuda") for _ in range(3))
    K, V, q = c.k.cuda(), c.v.cuda(), q.cuda()
    for b, (h, n) in enumerate(zip(c.held, c.new)):
        if n == 0:
            continue
        p = torch.arange(h + n)
        rows = c.table[b].long()[p // c.page]
        ok = torch.tensor([int(r) not in missing and 0 <= int(r) < c.n_pages for r in rows])
        rows, slot = torch.where(ok, rows, 0).cuda(), (p % c.page).cuda()
        k, v = K[rows, :, slot].double(), V[rows, :, slot].double()
        k[~ok.cuda()], v[~ok.cuda()] = 0.0, 0.0
        qs = q[c.start[b]:c.start[b] + n].double().view(n, c.G, share, c.D)
        s = torch.einsum("tgsd,jgd->gstj", qs, k) * scale
        big = torch.einsum("tgsd,jgd->gstj", qs.abs(), k.abs()) * abs(scale)
        if cap:
            s = cap * torch.tanh(s / cap)
        seen = (p[None] <= h + torch.arange(n)[:, None]).cuda() & ok.cuda()[None]
        s = s.masked_fill(~seen, -math.inf)
        w = torch.softmax(s, -1)
        at = slice(c.start[b], c.start[b] + n)
        out[at] = torch.einsum("gstj,jgd->tgsd", w, v).reshape(n, c.H, c.D)
        size[at] = torch.einsum("gstj,jgd->tgsd", w, v.abs()).reshape(n, c.H, c.D)
        top[at] = big.masked_fill(~seen, 0.0).amax(-1).permute(2, 0, 1).reshape(n, c.H)[..., None]
    return out, size, top


def tolerance(c, want, size, top, cap):
    """The result's rounding; of the weights (relative to sum w |v|): their rounding for the tensor cores (half a step of the cache's type, 2^-21 where they are the
    sum of two fp16 numbers), what scores are off by (dim + 8 roundings of 2^-24 of sum |q k|, with fp32 queries 2^-21 of it from their split; a cap: 2^-20 of it), exponentials 2^-21."""
    one = HALF_STEP[c.act] if c.act != "f32" else 2.0 ** -21
    score = ((c.D + 8) * 2.0 ** -24 + (2.0 ** -21 if c.act == "f32" else 0)) * top + 2.0 ** -20 * cap
    return HALF_STEP[c.act] * want.abs() + (one + 2.0 ** -21 + 2 * score) * size + (2.0 ** -25 if c.act == "f16" else 0)


def attention_case(lib, H, G, D, act, kv, page, held, new, cap=0.0, scale=None, seed=0, ragged=None, joint=False, pad=0, in_place=False, slack=0, shared=(), groups=None, sharp=1.0,
                   stream=None):
    c = Cache(H, G, D, act, kv, page, held, new, seed, ragged, joint, shared)
    c.fill(scale=sharp)
    scale = 1.2 / math.sqrt(D) if scale is None else scale
    T, ld = c.tokens + pad, H * D + slack
    q = torch.randn(T, ld, generator=c.gen).to(TYPES[act][0])
    d = q.cuda()
    o = d if in_place else torch.full((T, H * D + 8), 9.0, dtype=d.dtype, device="cuda")
    before, desc, g = o.clone(), c.upload(), None
    if groups is None and shared:
        groups = ([first for first, _, _ in shared] + [shared[-1][1]], [pages for _, _, pages in shared])
    if groups:
        starts, pages = i32(groups[0]), i32(groups[1])
        g = capi.PagedGroups(len(groups[1]), starts.data_ptr(), pages.data_ptr())
        torch.cuda.synchronize()
    want, size, top = attention_oracle(c, q[:c.tokens, :H * D], scale, cap)
    torch.cuda.synchronize()
    done(lib, lib.bpd_paged_attention_cuda(desc, d.data_ptr(), ld, o.data_ptr(), o.stride(0), T, scale, cap, None if g is None else C.byref(g), stream))
    got = o[:c.tokens, :H * D].double().view(c.tokens, H, D)
    miss = (got - want).abs() - tolerance(c, want, size, top, cap)
    assert torch.isfinite(got).all()
    worst = miss.amax().item() if miss.numel() else -1.0
    assert worst <= 0, (worst, [int(i) for i in np.unravel_index(int(miss.argmax()), tuple(miss.shape))])
    assert torch.equal(o[c.tokens:], before[c.tokens:]) and torch.equal(o[:, H * D:], before[:, H * D:])
    return o[:c.tokens, :H * D].clone()


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("H,G,D,page", [(4, 2, 64, 16), (3, 3, 128, 8), (8, 1, 96, 32), (14, 2, 64, 128), (2, 1, 80, 16), (6, 2, 8, 256), (32, 8, 128, 16), (16, 1, 128, 16), (24, 2, 56, 64)])
def test_one_token(lib, act, kv, H, G, D, page):
    attention_case(lib, H, G, D, act, kv, page, [0, 1, 7, 15, 16, 31, 200, 1000], [1] * 8, seed=D)


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("held", [[4000], [127], [128], [129], [0], [5000, 3], [0] * 5, [300] * 40])
def test_one_token_lengths(lib, act, kv, held):
    attention_case(lib, 8, 2, 128, act, kv, 16, held, [1] * len(held), seed=len(held))


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("H,G,D,page", [(4, 2, 64, 16), (3, 3, 128, 8), (8, 1, 96, 32), (2, 1, 80, 256), (32, 8, 128, 16), (14, 2, 64, 128), (5, 1, 128, 16)])
def test_prompts(lib, act, kv, H, G, D, page):
    attention_case(lib, H, G, D, act, kv, page, [0, 0, 100, 513, 0], [1, 130, 3, 300, 65], seed=D)


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("held,new", [([0], [128]), ([0], [129]), ([1], [127]), ([1000], [64]), ([0], [700]), ([37] * 6, [17, 0, 33, 1, 0, 2]), ([10] * 30 + [0], [1] * 30 + [500])])
def test_portions(lib, act, kv, held, new):
    attention_case(lib, 8, 2, 128, act, kv, 16, held, new, seed=len(new), pad=2)


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("cap", [0.5, 30.0])
def test_caps(lib, act, kv, cap):
    attention_case(lib, 8, 2, 64, act, kv, 16, [3, 500, 0, 60], [1, 1, 1, 1], cap=cap, scale=1.0)
    attention_case(lib, 8, 2, 128, act, kv, 16, [3, 500, 0, 60], [1, 40, 200, 2], cap=cap, scale=1.0)


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_scales(lib, act, kv, scale):
    """Every position alike, the other sign, and scores so far apart that one position takes all."""
    attention_case(lib, 4, 1, 64, act, kv, 16, [700, 30], [1, 1], scale=scale)
    attention_case(lib, 4, 1, 64, act, kv, 16, [700, 30], [50, 140], scale=scale)


@pytest.mark.parametrize("act,kv", PAIRS)
def test_forms(lib, act, kv):
    """In place, strides, pools in one block, bounds where every sequence brings one token, spare rows."""
    for i, form in enumerate([dict(in_place=True), dict(slack=16), dict(joint=True), dict(ragged=True), dict(pad=5), dict(ragged=True, pad=2, in_place=True, slack=8)]):
        attention_case(lib, 6, 2, 64, act, kv, 16, [5, 400, 100], [1, 1, 1], seed=i, **form)
        attention_case(lib, 6, 2, 64, act, kv, 16, [5, 400, 100], [70, 1, 30], seed=i, **{k: v for k, v in form.items() if k != "ragged"})


SHARED = [
    # (held, new, ranges that share pages of 16)
    ([100, 96, 130], [1, 1, 1], [(0, 3, 6)]),
    ([1000] * 9, [1] * 9, [(0, 9, 62)]),
    ([1000] * 40, [1] * 40, [(0, 40, 60)]),
    ([64, 64, 700, 705, 710, 5], [1] * 6, [(0, 2, 4), (2, 5, 43)]),
    ([64, 64, 700, 705, 710, 5, 9], [1, 2, 1, 30, 3, 1, 4], [(0, 2, 4), (2, 5, 43)]),
    ([512] * 5, [100, 1, 0, 33, 7], [(0, 5, 32)]),
    ([320, 320, 400], [1, 1, 1], [(0, 2, 20), (2, 3, 25)]),            # nothing of its own but the new token; a group of one
    ([50, 50], [1, 1], [(0, 2, 0)]),
]


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("held,new,shared", SHARED, ids=str)
def test_shared_prefixes(lib, act, kv, held, new, shared):
    for H, G, D in ((8, 2, 128), (6, 6, 64), (8, 1, 80)):
        with_groups = attention_case(lib, H, G, D, act, kv, 16, held, new, shared=shared, pad=1)
        without = attention_case(lib, H, G, D, act, kv, 16, held, new, shared=shared, groups=([0], []), pad=1)
        assert (with_groups.float() - without.float()).abs().max() <= 0.02


@pytest.mark.parametrize("act,kv", PAIRS)
def test_groups_leave_sequences_out(lib, act, kv):
    """Sequences ahead of the first group and behind the last one share nothing."""
    attention_case(lib, 4, 2, 64, act, kv, 16, [200, 300, 300, 300, 20], [1] * 5, shared=[(1, 4, 15)])
    attention_case(lib, 4, 2, 64, act, kv, 16, [200, 300, 300, 300, 20], [3, 1, 40, 2, 9], shared=[(1, 4, 15)], cap=20.0)


def test_groups_that_claim_too_much(lib):
    """A prefix longer than a member holds ends where that member's positions end: the rest is each one's own."""
    attention_case(lib, 4, 2, 64, "bf16", "bf16", 16, [40, 300, 300], [1] * 3, shared=[(0, 3, 2)], groups=([0, 3], [1000]))
    attention_case(lib, 4, 2, 64, "bf16", "bf16", 16, [40, 300, 300], [1] * 3, shared=[(0, 3, 2)], groups=([0, 3], [-5]))


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 1, 20, 3]])
def test_bad_pages_and_lengths(lib, new):
    """Pages that the pool does not have take no part, a sequence whose length makes no sense is left out, and the status says so."""
    c = Cache(4, 2, 64, "bf16", "bf16", 16, [100, 60, 200, 30], new, 3)
    c.fill()
    c.table[0, 2], c.table[2, 0], c.table[2, 5] = -1, c.n_pages, 2 ** 31 - 1
    q = torch.randn(c.tokens, 4 * 64, generator=c.gen).bfloat16()
    want, size, top = attention_oracle(c, q, 0.1, 0.0)
    c.held[3] = -4
    desc = c.upload()
    d, o = q.cuda(), torch.full((c.tokens, 256), 9.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    assert lib.bpd_paged_attention_cuda(desc, d.data_ptr(), 256, o.data_ptr(), 256, c.tokens, 0.1, 0.0, None, None) == 0
    torch.cuda.synchronize()
    assert lib.bpdq_last_status() == -4
    lib.bpdq_clear_status()
    n = c.start[3]
    assert (o[n:] == 9.0).all()
    miss = (o[:n].double().view(n, 4, 64) - want[:n]).abs() - tolerance(c, want, size, top, 0.0)[:n]
    assert miss.max() <= 0


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (4, 2, 64)])
@pytest.mark.parametrize("held,new", [([100, 100, 30], [1, 1, 1]), ([100, 60, 30], [90, 3, 200])])
def test_a_key_without_a_number(lib, act, kv, H, G, D, held, new):
    """A NaN among the keys shows in the rows that see it, wherever it lies in a block, and in no others."""
    for place in (70, 71, 72, 73, 74, 75, 76, 77, 100):
        c = Cache(H, G, D, act, kv, 16, held, new, place)
        c.fill()
        clean = c.k.clone()
        c.k[c.table[0, place // 16].long(), 1, place % 16, 5] = float("nan")
        q = torch.randn(c.tokens, H * D, generator=c.gen).to(TYPES[act][0])
        desc, d, o = c.upload(), q.cuda(), torch.full((c.tokens, H * D), 9.0, dtype=TYPES[act][0], device="cuda")
        torch.cuda.synchronize()
        done(lib, lib.bpd_paged_attention_cuda(desc, d.data_ptr(), H * D, o.data_ptr(), H * D, c.tokens, 0.1, 0.0, None, None))
        c.k.copy_(clean)
        want, size, top = attention_oracle(c, q, 0.1, 0.0)
        got = o.double().view(c.tokens, H, D)
        sees = torch.zeros(c.tokens, H, dtype=torch.bool)
        for t in range(new[0]):
            sees[t, H // G:] = held[0] + t >= place
        sees = sees.cuda()
        assert torch.isnan(got[sees]).all()
        assert ((got - want).abs() <= tolerance(c, want, size, top, 0.0))[~sees].all()


@pytest.mark.parametrize("starts", [[0, 10, 5, 8, 12], [0, 10, 5, 12, 11], [3, 1, 12, 0, 12], [0, 12, 0, 12, 0]])
def test_bounds_that_run_backwards_inside_a_group(lib, starts):
    """What makes no sense is passed over and reported, and the next call is right."""
    c = Cache(4, 2, 64, "bf16", "bf16", 16, [100, 96, 130, 100], [3, 3, 3, 3], 9, shared=[(0, 4, 6)])
    c.fill()
    desc = c.upload()
    q = torch.randn(12, 256, generator=c.gen).bfloat16()
    want, size, top = attention_oracle(c, q, 0.1, 0.0)
    bounds, pages = i32([0, 4]), i32([6])
    g = C.byref(capi.PagedGroups(1, bounds.data_ptr(), pages.data_ptr()))
    d, o = q.cuda(), torch.zeros(12, 256, dtype=torch.bfloat16, device="cuda")
    right = c.d_start.clone()
    c.d_start.copy_(i32(starts))
    torch.cuda.synchronize()
    assert lib.bpd_paged_attention_cuda(desc, d.data_ptr(), 256, o.data_ptr(), 256, 12, 0.1, 0.0, g, None) == 0
    torch.cuda.synchronize()
    assert lib.bpdq_last_status() == -4
    lib.bpdq_clear_status()
    c.d_start.copy_(right)
    torch.cuda.synchronize()
    done(lib, lib.bpd_paged_attention_cuda(desc, d.data_ptr(), 256, o.data_ptr(), 256, 12, 0.1, 0.0, g, None))
    assert ((o.double().view(12, 4, 64) - want).abs() <= tolerance(c, want, size, top, 0.0)).all()


def test_a_sequence_without_a_page_is_zero(lib):
    c = Cache(4, 2, 64, "bf16", "bf16", 16, [20, 20], [1, 1], 3)
    c.fill()
    c.table[0, :] = -1
    desc = c.upload()
    d, o = torch.randn(2, 256).bfloat16().cuda(), torch.full((2, 256), 9.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    assert lib.bpd_paged_attention_cuda(desc, d.data_ptr(), 256, o.data_ptr(), 256, 2, 0.1, 0.0, None, None) == 0
    torch.cuda.synchronize()
    assert lib.bpdq_last_status() == -4
    lib.bpdq_clear_status()
    assert (o[0] == 0).all() and torch.isfinite(o[1]).all() and (o[1] != 9.0).any()


def test_cache_beyond_four_gigabytes(lib):
    """Pages whose offsets pass 32 bits, in elements too."""
    G, page, D = 8, 256, 128
    n_pages = 2 ** 32 // (G * page * D) + 40
    k = torch.zeros(n_pages, G, page, D, dtype=torch.bfloat16, device="cuda")
    held, g = [700, 300], torch.Generator(device="cuda").manual_seed(1)
    table = torch.tensor([[n_pages - 1, n_pages - 7, 3], [n_pages - 20, n_pages - 3, 0]], dtype=torch.int32)
    q = torch.randn(2, 32, D, device="cuda", generator=g).bfloat16()
    x = torch.randn(2, 2 * G, D, device="cuda", generator=g).bfloat16()
    for r in table.flatten().tolist():
        k[r] = torch.randn(G, page, D, device="cuda", generator=g).bfloat16()
    d_table, d_len = table.cuda(), i32(held)
    kv = capi.PagedKv(32, G, D, 2, 2, page, n_pages, 2, 3, 0, k.data_ptr(), k.data_ptr(), d_table.data_ptr(), d_len.data_ptr(), None)     # values are the keys
    o = torch.empty(2, 32, D, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    done(lib, lib.bpd_paged_append_cuda(C.byref(kv), None, 0, None, 0, x.data_ptr(), 2 * G * D, x.data_ptr(), 2 * G * D, 2, 0, 0, None, None))
    for b, h in enumerate(held):
        assert torch.equal(k[table[b, h // page].item(), :, h % page], x[b, :G])
    done(lib, lib.bpd_paged_attention_cuda(C.byref(kv), q.data_ptr(), 32 * D, o.data_ptr(), 32 * D, 2, 0.09, 0.0, None, None))
    for b, h in enumerate(held):
        p = torch.arange(h + 1, device="cuda")
        keys = k[d_table[b].long()[p // page], :, p % page].double()
        w = torch.softmax(torch.einsum("gsd,jgd->gsj", q[b].double().view(G, 4, D), keys) * 0.09, -1)
        want, size = torch.einsum("gsj,jgd->gsd", w, keys).reshape(32, D), torch.einsum("gsj,jgd->gsd", w, keys.abs()).reshape(32, D)
        assert ((o[b].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 1e-4) * size).all()


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("H,G,D", [(34, 2, 64), (32, 1, 128), (128, 1, 128), (128, 1, 64), (200, 2, 40)])
def test_many_heads_on_a_key_head(lib, act, kv, H, G, D):
    """More rows per token than the kernel for few takes, up to a whole tile; shares that leave a tile's last rows empty."""
    attention_case(lib, H, G, D, act, kv, 16, [0, 5, 300, 64], [1] * 4, seed=H)
    attention_case(lib, H, G, D, act, kv, 16, [0, 5, 300, 64], [9, 1, 2, 30], seed=H, pad=1)
    attention_case(lib, H, G, D, act, kv, 16, [200, 200, 230], [1, 2, 1], shared=[(0, 3, 12)], seed=H)


@pytest.mark.parametrize("B,held,new", [(1, 6000, 300), (1, 200, 3000), (60, 6000, 1)])
def test_long_sums_of_fp32(lib, B, held, new):
    """The tensor pipe cuts its sums off toward zero, which adds up where values have one sign.  At most 32 sums follow one another (256 keys, by sixteen, the
    weights in two parts), each less than one step of fp32 short (2^-23 of it; half a step would be right for rounding, not for cutting off), of a sum that grows
    evenly to its whole: (1 + 2 + .. + 32) / 32 * 2^-23 = 1.04 * 2^-19; and what scores and weights are off by: 2^-21 (scores of unit size, cut off 16 times, 16 * 2^-25).
    In one go, without that limit, the 6300 keys would be 394 sums of a stream: up to 2^-15."""
    c = Cache(8, 2, 128, "f32", "f16", 16, [held] * B, [new] * B, 3)
    c.fill()
    c.v.abs_()
    q = torch.randn(c.tokens, 1024, generator=c.gen)
    d, desc = q.cuda(), c.upload()
    o = torch.empty_like(d)
    torch.cuda.synchronize()
    done(lib, lib.bpd_paged_attention_cuda(desc, d.data_ptr(), 1024, o.data_ptr(), 1024, c.tokens, 0.09, 0.0, None, None))
    want = attention_oracle(c, q, 0.09, 0.0)[0]
    error = o.double().view(c.tokens, 8, 128) - want
    assert error.norm() <= (1.04 * 2.0 ** -19 + 2.0 ** -21) * want.norm()
    assert abs((error * want).sum()) <= (1.04 * 2.0 ** -19 + 2.0 ** -21) * (want * want).sum()


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("H,G,new", [(16, 4, [4] * 7), (16, 4, [4, 3, 2, 4, 1, 0, 4]), (16, 2, [2] * 7), (16, 2, [2, 1, 2, 2, 1, 1, 2]), (4, 4, [16, 9, 12, 10, 16, 11, 13]), (6, 2, [5, 3, 4, 5, 4, 5, 3])])
def test_a_few_tokens_each(lib, act, kv, H, G, new):
    """Guessed tokens checked in one step: nine to sixteen rows of a sequence."""
    held = [0, 1, 15, 400, 2000, 33, 127]
    attention_case(lib, H, G, 128, act, kv, 16, held, new, seed=H, ragged=True)
    attention_case(lib, H, G, 64, act, kv, 32, held, new, seed=H, ragged=True, cap=15.0, pad=3)
    attention_case(lib, H, G, 128, act, kv, 16, [500] * 7, new, seed=H, ragged=True, shared=[(0, 3, 20), (3, 7, 31)])


@pytest.mark.parametrize("page", [8, 32, 64, 128, 256])
@pytest.mark.parametrize("act,kv", PAIRS)
def test_page_sizes(lib, act, kv, page):
    """Pages smaller and larger than a block of keys, shared ones among them, which a block may begin inside."""
    n = 512 // page
    for H, G, D in ((8, 2, 128), (4, 1, 72)):
        attention_case(lib, H, G, D, act, kv, page, [512 + 9, 512, 700, 600], [1] * 4, shared=[(0, 4, n)], seed=page)
        attention_case(lib, H, G, D, act, kv, page, [512 + 9, 512, 700, 600, 0], [1, 70, 300, 2, 260], shared=[(0, 4, n)], seed=page)


@pytest.mark.parametrize("batch,sets", [(1280, 0), (1000, 280), (1278, 2)])
def test_as_many_sequences_as_there_may_be(lib, batch, sets):
    """With one token each, and with a long prompt among them."""
    gen = torch.Generator().manual_seed(batch)
    held = (torch.randint(0, 60, (batch,), generator=gen) + 16).tolist()
    shared = [(batch * i // sets, batch * (i + 1) // sets, 1) for i in range(sets)]
    attention_case(lib, 4, 2, 64, "bf16", "bf16", 16, held, [1] * batch, shared=shared)
    new = [1] * batch
    new[batch // 3] = 200
    new[batch // 2] = 0
    attention_case(lib, 4, 2, 64, "bf16", "bf16", 16, held, new, shared=shared)


# ---- workspaces, streams, recordings

@pytest.mark.parametrize("new", [[1] * 6, [1, 40, 1, 300, 2, 1]])
def test_own_scratch_and_recordings(lib, new):
    """The form with the caller's scratch, on a stream, recorded, replayed after lengths, tables and queries have changed, gives the same bits as plain calls."""
    c = Cache(8, 2, 128, "bf16", "bf16", 16, [900, 40, 7, 320, 1500, 64], new, 5, spare_entries=9)
    c.table = torch.arange(len(new) * c.max_pages, dtype=torch.int32).view(len(new), -1)
    c.n_pages = c.table.numel()
    c.pool = torch.randn(2, c.n_pages, 2, 16, 128, generator=c.gen).bfloat16()
    c.k, c.v = c.pool[0], c.pool[1]
    desc = c.upload()
    bounds, pages = i32([0, 3, 6]), i32([0, 4])
    g = C.byref(capi.PagedGroups(2, bounds.data_ptr(), pages.data_ptr()))
    q = torch.randn(c.tokens, 8 * 128, generator=c.gen).bfloat16().cuda()
    size = lib.bpdq_paged_attention_workspace_bytes(desc, c.tokens, g)
    assert size > 0
    ws, o = torch.empty(size, dtype=torch.uint8, device="cuda").fill_(255), torch.empty_like(q)
    s = lib.bpdq_stream_create()
    torch.cuda.synchronize()

    def call(out, ws_ptr, stream):
        if ws_ptr is None:
            return lib.bpd_paged_attention_cuda(desc, q.data_ptr(), 1024, out.data_ptr(), 1024, c.tokens, 0.1, 0.0, g, stream)
        return lib.bpd_paged_attention_ws_cuda(desc, q.data_ptr(), 1024, out.data_ptr(), 1024, c.tokens, 0.1, 0.0, g, ws_ptr, size, stream)

    assert lib.bpdq_graph_begin(s) == 0
    assert call(o, ws.data_ptr(), s) == 0
    rec = lib.bpdq_graph_end(s)
    assert rec
    for i in range(3):
        o.fill_(9.0)
        if i:
            q.mul_(0.7)
            c.d_len.add_(i32([17, 0, 3, 100, 5, 31]))
            c.d_table.copy_(c.d_table.roll(1, 1))
            c.d_table[4:, :4] = c.d_table[3, :4]
        else:
            c.d_table[4:, :4] = c.d_table[3, :4]
        torch.cuda.synchronize()
        assert lib.bpdq_graph_launch(rec, s) == 0 and lib.bpdq_stream_sync(s) == 0
        want = torch.empty_like(q)
        assert call(want, None, None) == 0
        torch.cuda.synchronize()
        assert torch.equal(o, want), i
    assert lib.bpdq_last_status() == 0
    assert lib.bpd_paged_attention_ws_cuda(desc, q.data_ptr(), 1024, o.data_ptr(), 1024, c.tokens, 0.1, 0.0, g, ws.data_ptr(), size - 1, None) in (0, -3)
    torch.cuda.synchronize()
    lib.bpdq_clear_status()
    lib.bpdq_graph_destroy(rec)
    lib.bpdq_stream_destroy(s)


@pytest.mark.parametrize("new", [[1] * 5, [1, 150, 1, 33, 4]])
def test_two_at_once(lib, new):
    """Two streams' recordings, each with its scratch, side by side and again and again, give what each gives alone."""
    runs = []
    for i in range(2):
        c = Cache(8, 2, 128, "bf16", "bf16", 16, [800 + 300 * i, 0, 777, 63, 2000], new, 20 + i)
        c.fill()
        q = torch.randn(c.tokens, 1024, generator=c.gen).bfloat16().cuda()
        desc = c.upload()
        size = lib.bpdq_paged_attention_workspace_bytes(desc, c.tokens, None)
        ws, o = torch.empty(size, dtype=torch.uint8, device="cuda").fill_(255), torch.full_like(q, 9.0)
        want = torch.empty_like(q)
        torch.cuda.synchronize()
        done(lib, lib.bpd_paged_attention_cuda(desc, q.data_ptr(), 1024, want.data_ptr(), 1024, c.tokens, 0.1, 0.0, None, None))
        stream = lib.bpdq_stream_create()
        assert lib.bpdq_graph_begin(stream) == 0
        for _ in range(5):
            assert lib.bpd_paged_attention_ws_cuda(desc, q.data_ptr(), 1024, o.data_ptr(), 1024, c.tokens, 0.1, 0.0, None, ws.data_ptr(), size, stream) == 0
        rec = lib.bpdq_graph_end(stream)
        assert rec
        runs.append((c, q, desc, ws, o, want, stream, rec))
    for _ in range(20):
        for *_, stream, rec in runs:
            assert lib.bpdq_graph_launch(rec, stream) == 0
    for c, q, desc, ws, o, want, stream, rec in runs:
        assert lib.bpdq_stream_sync(stream) == 0
    torch.cuda.synchronize()
    assert lib.bpdq_last_status() == 0
    for c, q, desc, ws, o, want, stream, rec in runs:
        assert torch.equal(o, want)
        lib.bpdq_graph_destroy(rec)
        lib.bpdq_stream_destroy(stream)


# ---- together

def test_a_batch_decodes(lib):
    """Two layers' worth of steps as a server makes them: prompts in a portion, then tokens, appended, attended and sampled, against attention over
    the whole sequences in 64 bits; two sequences begin alike and share pages."""
    H, G, D, page, vocab, steps = 8, 2, 64, 16, 500, 6
    gen = torch.Generator().manual_seed(7)
    embed, head = torch.randn(vocab, (H + 2 * G) * D, generator=gen), torch.randn(H * D, vocab, generator=gen) / math.sqrt(H * D) * 4
    freq = (10000.0 ** (-torch.arange(D // 2).double() / (D // 2))).float()
    prompts = [torch.randint(0, vocab, (n,), generator=gen).tolist() for n in (70, 70, 5)]
    prompts[1][:64] = prompts[0][:64]                       # four whole pages
    max_pages, B = 8, 3
    table = torch.arange(B * max_pages, dtype=torch.int32).view(B, max_pages)
    table[1, :4] = table[0, :4]
    pool = torch.full((2, B * max_pages, G, page, D), float("nan"), dtype=torch.float16, device="cuda")
    d_table, d_len, d_embed, d_head, d_freq = table.cuda(), i32([0, 64, 0]), embed.cuda(), head.cuda(), freq.cuda()
    bounds, pages = i32([0, 2]), i32([4])
    shared = capi.PagedGroups(1, bounds.data_ptr(), pages.data_ptr())
    u = torch.rand(steps, B, generator=gen)
    t, k, p = torch.tensor([0.8, 1.0, 0.0], device="cuda"), i32([40, 0, 0]), torch.tensor([0.9, 0.95, 1.0], device="cuda")
    sequences = [list(q) for q in prompts]
    fed = [0, 64, 0]                                        # the second sequence's pages are the first one's: it brings what follows
    for step in range(steps):
        new = [len(s) - f for s, f in zip(sequences, fed)]
        starts = [0, new[0], new[0] + new[1], sum(new)]
        d_start = i32(starts)
        ids = torch.tensor([x for s, f in zip(sequences, fed) for x in s[f:]])
        qkv = d_embed[ids.cuda()].contiguous()
        ld, T = qkv.stride(0), len(ids)
        kv = capi.PagedKv(H, G, D, 0, 1, page, B * max_pages, B, max_pages, 0, pool[0].data_ptr(), pool[1].data_ptr(), d_table.data_ptr(), d_len.data_ptr(),
                          None if new == [1] * B else d_start.data_ptr())
        torch.cuda.synchronize()
        x = qkv.data_ptr()
        assert lib.bpd_paged_append_cuda(C.byref(kv), x, ld, x, ld, x + H * D * 4, ld, x + (H + G) * D * 4, ld, T, D, 1, d_freq.data_ptr(), None) == 0
        o = torch.empty(T, H * D, device="cuda")
        groups = C.byref(shared) if step else None           # the first step fills the shared pages
        done(lib, lib.bpd_paged_attention_cuda(C.byref(kv), x, ld, o.data_ptr(), H * D, T, D ** -0.5, 0.0, groups, None))
        last = torch.tensor(starts[1:], device="cuda") - 1
        logits = (o[last] @ d_head).contiguous()
        token = torch.empty(B, dtype=torch.int64, device="cuda")
        du = u[step].cuda()
        torch.cuda.synchronize()
        done(lib, lib.bpd_sample_cuda(logits.data_ptr(), 0, vocab, B, vocab, t.data_ptr(), k.data_ptr(), p.data_ptr(), None, du.data_ptr(), token.data_ptr(), None, None))
        for b, s in enumerate(sequences):
            y = embed[torch.tensor(s)].double().view(len(s), -1, D)
            z = turned(y[:, :H + G], torch.arange(len(s)), D, 1, freq)
            key, value = z[:, H:].half().double(), y[:, H + G:].half().double()
            w = torch.softmax(torch.einsum("gsd,jgd->gsj", z[-1, :H].view(G, H // G, D), key) * D ** -0.5, -1)
            want = torch.einsum("gsj,jgd->gsd", w, value).reshape(-1)
            # keys near a border of fp16 may be rounded to its other side: half a step more of them, scores of |q||k| / 8 <= 8 * 2^-11 each
            assert (o[last[b]].cpu().double() - want).abs().max() <= 0.01, (step, b)
        fed = [len(s) for s in sequences]
        d_len = i32(fed)
        for s, x in zip(sequences, token.cpu().tolist()):
            assert 0 <= x < vocab
            s.append(x)
        if step == 0:
            assert sequences[2][-1] == int(logits[2].argmax())


# ---- rows in which one position takes nearly all

def one_that_takes_nearly_all(c, gap, place, value):
    """Every sequence's position `place` (the last one, where there are fewer) scores `gap`, all others 0, exactly; it has the value given, the others positive ones."""
    c.fill()
    c.v.abs_()
    for b, (h, n) in enumerate(zip(c.held, c.new)):
        p = torch.arange(h + n)
        rows = c.table[b].long()[p // c.page]
        c.k[rows, :, p % c.page] = 0
        p = min(place, h)
        c.k[c.table[b, p // c.page].long(), :, p % c.page, 0] = gap
        c.v[c.table[b, p // c.page].long(), :, p % c.page] = value
    q = torch.randn(c.tokens, c.H, c.D, generator=c.gen)
    q[..., 0] = 1.0
    return q.reshape(c.tokens, -1).to(TYPES[c.act][0])


SMALL = [
    # (H, G, D, held, new, ranges that share pages): the kernel for few rows with one product and with two, the one for many, both in a call
    (8, 2, 128, [4000, 16000, 700], [1, 1, 1], ()),
    (8, 2, 64, [4000, 9000], [4, 4], ()),
    (4, 2, 128, [3000, 9000], [70, 100], ()),
    (4, 4, 64, [3000, 9000], [140, 1], ()),
    (8, 2, 128, [8000] * 9, [1] * 9, [(0, 9, 490)]),
]


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("gap", [11.0, 14.0, 17.5, 20.0])
@pytest.mark.parametrize("place", [0, 2500])
@pytest.mark.parametrize("value", [0.0, 1.0])
def test_small_weights(lib, act, kv, gap, place, value):
    """Weights far below the largest, thousands of them, are not lost.  With fp32 activations: 5e-6 of sum w |v|, 2^-36 of the largest weight on each, three roundings of the
    score (2^-24 of it each) and of the result.  16-bit types: weights rounded to half a step of the cache's type, of fp16 and 2^-32 of the largest."""
    for H, G, D, held, new, shared in SMALL:
        c = Cache(H, G, D, act, kv, 16, held, new, 5, shared=shared)
        q = one_that_takes_nearly_all(c, gap, place, value)
        desc, d = c.upload(), q.cuda()
        o = torch.full_like(d, 9.0)
        g = None
        if shared:
            starts, pages = i32([first for first, _, _ in shared] + [shared[-1][1]]), i32([n for _, _, n in shared])
            g = C.byref(capi.PagedGroups(len(shared), starts.data_ptr(), pages.data_ptr()))
        want, size, _ = attention_oracle(c, q, 1.0, 0.0)
        total = torch.zeros_like(want)
        for b, (h, n) in enumerate(zip(c.held, c.new)):
            p = torch.arange(h + n)
            total[c.start[b]:c.start[b] + n] = c.v[c.table[b].long()[p // 16], :, p % 16].double().sum(0).repeat_interleave(H // G, 0).cuda()
        done(lib, lib.bpd_paged_attention_cuda(desc, d.data_ptr(), H * D, o.data_ptr(), H * D, c.tokens, 1.0, 0.0, g, None))
        part = {"f32": 5e-6, "f16": 2.0 ** -11 + 2.0 ** -20, "bf16": 2.0 ** -8 + 2.0 ** -20}[act] + 2 * 3 * 2.0 ** -24 * gap
        floor = {"f32": 2.0 ** -36, "f16": 2.0 ** -32, "bf16": 0.0}[act]
        bound = HALF_STEP[act] * want + part * size + floor * total + (2.0 ** -25 if act == "f16" else 0)
        worst = ((o.double().view_as(want) - want).abs() / bound).amax().item()
        assert worst <= 1, (H, G, D, worst)


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("row", ["cleared", "another's", "short"])
@pytest.mark.parametrize("new", [[0, 1, 1, 1], [0, 30, 1, 200], [0, 0, 1, 1], [0, 0, 0, 5]])
def test_groups_whose_first_sequence_brings_nothing(lib, act, kv, row, new):
    """A slot whose sequence is finished: its row of the table is not what the others share."""
    held = [0, 640, 700, 655]
    for H, G, D in ((8, 2, 128), (4, 4, 64)):
        c = Cache(H, G, D, act, kv, 16, held, new, 7, ragged=True, shared=[(1, 4, 40)])
        if row != "cleared":
            c.table[0] = torch.randint(0, c.n_pages, (c.max_pages,), generator=c.gen, dtype=torch.int32)
        c.held[0] = 5 if row == "short" else 0
        c.fill()
        q = torch.randn(c.tokens, H * D, generator=c.gen).to(TYPES[act][0])
        want, size, top = attention_oracle(c, q, 0.1, 0.0)
        bounds, pages = i32([0, 4]), i32([40])
        g = C.byref(capi.PagedGroups(1, bounds.data_ptr(), pages.data_ptr()))
        desc, d = c.upload(), q.cuda()
        o = torch.full_like(d, 9.0)
        done(lib, lib.bpd_paged_attention_cuda(desc, d.data_ptr(), H * D, o.data_ptr(), H * D, c.tokens, 0.1, 0.0, g, None))
        assert ((o.double().view_as(want) - want).abs() <= tolerance(c, want, size, top, 0.0)).all()


@pytest.mark.parametrize("act,kv", PAIRS)
def test_what_the_launches_before_have_written(lib, act, kv):
    """A step right behind what fills its cache, queries, lengths and table, prompts and single tokens in one call, again and again without a wait between: the bits
    that the same steps give one at a time."""
    H, G, D, new = 8, 2, 128, [1, 90, 1, 1, 200, 1]
    c = Cache(H, G, D, act, kv, 16, [700, 40, 3000, 95, 0, 16], new, 3, spare_entries=4)
    c.fill(everything=False)
    desc, T, ld = c.upload(), c.tokens, (H + 2 * G) * D
    rows = [torch.randn(T, ld, generator=c.gen).to(TYPES[act][0]).cuda() for _ in range(12)]
    lengths = [i32([max(0, h - 3 * i) for h in c.held]) for i in range(12)]
    tables = [c.d_table.clone() for _ in range(12)]
    for i, t in enumerate(tables):
        t[:, :1] = t[:, :1].roll(i, 0)
    x, out = torch.empty_like(rows[0]), [torch.empty(T, H * D, dtype=rows[0].dtype, device="cuda") for _ in range(24)]
    size, start = x.element_size(), c.d_pool.clone()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()

    def steps(at, wait):
        with torch.cuda.stream(stream):
            c.d_pool.copy_(start)
            for i in range(12):
                x.copy_(rows[i])
                c.d_len.copy_(lengths[i])
                c.d_table.copy_(tables[i])
                p, s = x.data_ptr(), stream.cuda_stream
                assert lib.bpd_paged_append_cuda(desc, p, ld, p, ld, p + H * D * size, ld, p + (H + G) * D * size, ld, T, 0, 0, None, s) == 0
                if wait:
                    stream.synchronize()
                assert lib.bpd_paged_attention_cuda(desc, p, ld, out[at + i].data_ptr(), H * D, T, 0.1, 0.0, None, s) == 0
                if wait:
                    stream.synchronize()
        stream.synchronize()

    steps(0, True)
    for _ in range(5):
        steps(12, False)
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(out[:12], out[12:]))
    assert lib.bpdq_last_status() == 0


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("cap", [1e-42, 1e-30, 1e-6, 100.0, 1e5, 1e8, 3e38])
def test_caps_far_from_the_scores(lib, act, kv, cap):
    """A cap far above the scores changes nothing, one far below makes all positions alike.  What scores are off by (dim + 8 roundings of sum |q k|, 2^-21 of it by the split of fp32
    queries) and 2^-20 of what the cap leaves of them."""
    for new in ([1, 1, 1], [60, 1, 150]):
        c = Cache(8, 2, 64, act, kv, 16, [3, 500, 60], new, 11)
        c.fill()
        q = torch.randn(c.tokens, 512, generator=c.gen).to(TYPES[act][0])
        want, size, top = attention_oracle(c, q, 0.5, cap)
        desc, d = c.upload(), q.cuda()
        o = torch.full_like(d, 9.0)
        done(lib, lib.bpd_paged_attention_cuda(desc, d.data_ptr(), 512, o.data_ptr(), 512, c.tokens, 0.5, cap, None, None))
        miss = (o.double().view_as(want) - want).abs() - tolerance(c, want, size, top * (1 + 2.0 ** -20 / (c.D * 2.0 ** -24)), 0.0)
        assert miss.max() <= 0, (new, miss.max().item())


@pytest.mark.parametrize("new", [[1] * 4, [1, 90, 1, 20]])
def test_workspaces_that_are_too_small(lib, new):
    """A call with less than it needs is refused and leaves its results alone; what the size query says is enough wherever the workspace begins (16-byte aligned)."""
    c = Cache(8, 2, 128, "bf16", "bf16", 16, [300, 40, 1000, 64], new, 5)
    c.fill()
    q = torch.randn(c.tokens, 1024, generator=c.gen).bfloat16().cuda()
    desc = c.upload()
    size = lib.bpdq_paged_attention_workspace_bytes(desc, c.tokens, None)
    ws, o, want = torch.empty(size + 512, dtype=torch.uint8, device="cuda"), torch.full_like(q, 9.0), torch.empty_like(q)
    base = (ws.data_ptr() + 255) // 256 * 256
    torch.cuda.synchronize()

    def call(out, at, n):
        return lib.bpd_paged_attention_ws_cuda(desc, q.data_ptr(), 1024, out.data_ptr(), 1024, c.tokens, 0.1, 0.0, None, at, n, None)

    for at, n in ((base, size - 257), (base + 16, size - 17), (base, 16), (base, 0)):
        assert call(o, at, n) == -3
        torch.cuda.synchronize()
        assert lib.bpdq_last_status() == -3 and (o == 9.0).all()
        lib.bpdq_clear_status()
    done(lib, lib.bpd_paged_attention_cuda(desc, q.data_ptr(), 1024, want.data_ptr(), 1024, c.tokens, 0.1, 0.0, None, None))
    for at, n in ((base, size), (base, size - 256), (base + 16, size), (base + 240, size)):
        o.fill_(9.0)
        ws.fill_(255)
        torch.cuda.synchronize()
        done(lib, call(o, at, n))
        assert torch.equal(o, want)


@pytest.mark.parametrize("entry", [-1, -2, -3, -2 ** 31, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("act,kv", PAIRS)
def test_every_bad_page_is_reported(lib, act, kv, new, entry):
    """Whatever number stands in its place, to appending and to attention over few rows and many."""
    c = Cache(4, 2, 64, act, kv, 16, [100, 30], [new, new], 3, ragged=True)
    c.fill()
    c.table[0, 3] = entry
    q = torch.randn(c.tokens, 256, generator=c.gen).to(TYPES[act][0])
    want, size, top = attention_oracle(c, q, 0.1, 0.0)
    desc, d = c.upload(), q.cuda()
    o = torch.full_like(d, 9.0)
    torch.cuda.synchronize()
    assert lib.bpd_paged_attention_cuda(desc, d.data_ptr(), 256, o.data_ptr(), 256, c.tokens, 0.1, 0.0, None, None) == 0
    torch.cuda.synchronize()
    status = lib.bpdq_last_status()
    lib.bpdq_clear_status()
    assert status == -4
    assert ((o.double().view_as(want) - want).abs() <= tolerance(c, want, size, top, 0.0)).all()
    c.d_len[0] = 48                                          # the new tokens' first page is the bad one
    torch.cuda.synchronize()
    assert lib.bpd_paged_append_cuda(desc, None, 0, None, 0, d.data_ptr(), 256, d.data_ptr() + 128 * d.element_size(), 256, c.tokens, 0, 0, None, None) == 0
    torch.cuda.synchronize()
    status = lib.bpdq_last_status()
    lib.bpdq_clear_status()
    assert status == -4


@pytest.mark.parametrize("act,kv", PAIRS)
@pytest.mark.parametrize("new", [[1], [5], [70], [1, 300, 1]])
def test_a_long_context(lib, act, kv, new):
    """130 000 positions, for one token, a few, a portion, and a portion of a prompt beside it."""
    attention_case(lib, 8, 2, 128, act, kv, 32, [130000, 10, 900][:len(new)], new, seed=len(new), ragged=True)
