"""bpd_sample_cuda against its definition in 64 bits: the token has to be equal, whatever the cuts, the types and the shape of the row."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}
LOWEST = {"f32": torch.finfo(torch.float32).min, "f16": torch.finfo(torch.float16).min, "bf16": torch.finfo(torch.bfloat16).min}


def oracle(x, t, k, p, m, u):
    """(token, log probability) of one row; x float64, settings as fp32 numbers."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf
    if not t > 0:
        return int(x.argmax()), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(x == top, 0.0, (x - top) / t)
    z = np.where(np.isnan(z), -np.inf, z)               # finite numbers beside infinity
    w = np.exp(z)
    w[w < 2.0 ** -45] = 0.0                              # a part of the definition: such tokens are never chosen
    order = np.lexsort((np.arange(x.size), -x))         # by value, the lowest index first among equals
    order = order[x[order] > -np.inf]
    n = len(order)
    if k > 0:
        n = min(n, k)
    cum = np.cumsum(w[order[:n]])
    keep = n
    if p < 1:
        keep = min(keep, 1 + int((cum < p * cum[-1]).sum()))
    if m > 0:
        keep = min(keep, max(1, int((w[order[:n]] >= min(m, 1.0)).sum())))
    kept = np.sort(order[:keep])
    cum = np.cumsum(w[kept])
    u = min(max(u, 0.0), 1 - 2.0 ** -24)
    i = int((cum <= u * cum[-1]).sum())
    return int(kept[i]), z[kept[i]] - math.log(cum[-1])


def check(lib, x, kind, t=None, k=None, p=None, m=None, u=None, ld=None, stream=None, shift=0):
    """x: float32 [rows, vocab], rounded to the type here; settings: lists per row or None."""
    rows, vocab = x.shape
    ld = ld or vocab
    dtype, code = TYPES[kind]
    store = torch.full((rows * ld + shift,), float("nan"), dtype=dtype)
    at = store[shift:].view(rows, ld)
    at[:, :vocab] = torch.as_tensor(x).to(dtype)
    d = store.cuda()

    def dev(v, dtype):
        return None if v is None else torch.as_tensor(np.asarray(v), dtype=dtype, device="cuda")

    dt, dk, dp, dm = dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32), dev(m, torch.float32)
    u = [0.3] * rows if u is None else u
    du = dev(u, torch.float32)
    token, logp = torch.full((rows + 1,), -7, dtype=torch.int64, device="cuda"), torch.full((rows + 1,), 7.0, device="cuda")
    torch.cuda.synchronize()
    ptr = [None if v is None else v.data_ptr() for v in (dt, dk, dp, dm)]
    assert lib.bpd_sample_cuda(d.data_ptr() + shift * d.element_size(), code, ld, rows, vocab, *ptr, du.data_ptr(), token.data_ptr(), logp.data_ptr(), stream) == 0
    torch.cuda.synchronize()
    assert lib.bpdq_last_status() == 0
    token, logp = token.cpu().numpy(), logp.cpu().numpy()
    assert token[rows] == -7 and logp[rows] == 7.0
    exact = at[:, :vocab].double().numpy()

    def f(v, r, default):
        return default if v is None else float(np.float32(v[r]))

    for r in range(rows):
        want, lp = oracle(exact[r], f(t, r, 1.0), 0 if k is None else int(k[r]), f(p, r, 1.0), f(m, r, 0.0), f(u, r, 0.0))
        assert token[r] == want, (r, token[r], want)
        # fp32's rounding of the result, and 1e-12 of the sum
        assert logp[r] == lp or abs(logp[r] - lp) <= 2.0 ** -24 * abs(lp) + 1e-9, (r, logp[r], lp)
    return token[:rows]


def normal(rows, vocab, seed, scale=3.0):
    return (np.random.default_rng(seed).standard_normal((rows, vocab)) * scale).astype(np.float32)


SETTINGS = [dict(), dict(k=50), dict(p=0.9), dict(m=0.05), dict(k=40, p=0.95), dict(k=200, p=0.8, m=0.02), dict(p=0.99, m=0.01), dict(k=3000, p=0.97), dict(k=1), dict(p=1e-6), dict(m=1.0)]


def settings(rows, s):
    return {name: [v] * rows for name, v in s.items()}


@pytest.mark.parametrize("s", SETTINGS, ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (2, 33), (3, 1000), (2, 4097), (2, 32000), (1, 128256)])
def test_sizes(lib, rows, vocab, s):
    rng = np.random.default_rng(vocab)
    check(lib, normal(rows, vocab, vocab + 1), "f32", t=[0.8] * rows, u=rng.random(rows).astype(np.float32), **settings(rows, s))


@pytest.mark.parametrize("s", SETTINGS, ids=str)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_types_with_many_equal_values(lib, kind, s):
    rng = np.random.default_rng(5)
    for vocab, ld in ((5000, 5000), (8191, 8193), (32000, 32008)):
        check(lib, normal(3, vocab, vocab), kind, t=[1.0, 0.7, 1.5], u=rng.random(3).astype(np.float32), ld=ld, **settings(3, s))


@pytest.mark.parametrize("s", SETTINGS, ids=str)
def test_flat_rows(lib, s):
    """Rows of one value, of two, and nearly flat ones: far more elements at the cut than are sorted, equal ones decided by their index."""
    x = normal(5, 40000, 8, 0.01)
    x[0] = 1.25
    x[1] = np.where(np.arange(40000) % 3 == 0, 2.0, 1.0)
    x[2] = np.round(x[2] * 100) / 100
    check(lib, x, "f32", t=[1.0] * 5, u=[0.5, 0.999, 0.25, 0.75, 0.1], **settings(5, s))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("s", SETTINGS, ids=str)
def test_masked_rows(lib, kind, s):
    """Rows with -inf, NaN and the type's lowest value in masked places, with one place left, none left, and +inf."""
    vocab = 3001
    x = normal(9, vocab, 9)
    x[0, 5:] = -np.inf
    x[1, ::2] = np.nan
    x[2] = -np.inf
    x[3] = np.nan
    x[4] = -np.inf
    x[4, 2999] = -3.0
    x[5, 10:] = LOWEST[kind]
    x[6, [7, 1000, 2000]] = np.inf
    x[7] = LOWEST[kind]
    x[8, 0] = np.nan
    x[8, 1] = np.inf
    check(lib, x, kind, t=[0.9] * 9, u=[0.7] * 9, **settings(9, s))


@pytest.mark.parametrize("t", [0.0, -1.0, float("nan"), 1e-40, 1e-3, 0.01, 50.0, 1e6, 1e30, float("inf")])
@pytest.mark.parametrize("s", SETTINGS, ids=str)
def test_temperatures(lib, t, s):
    x = normal(3, 6000, 10)
    x[2, 17] = x[2].max()
    check(lib, x, "f32", t=[t] * 3, u=[0.0, 0.5, 0.999], **settings(3, s))


def test_settings_beyond_their_ranges(lib):
    x = normal(12, 2500, 11)
    check(lib, x, "f32", t=[1.0] * 12, k=[-1, 0, 2500, 2499, 10 ** 6, 1, 1024, 1025, 1023, 5, 5, 5], p=[1.0, 2.0, 0.0, -1.0, float("nan"), 0.5, 0.999999, 1 - 2.0 ** -24, 0.3, 0.5, 0.5, 0.5],
          m=[0.0, -1.0, float("nan"), 2.0, 1.0, 0.5, 1e-30, 1e-45, 0.0, 0.5, 0.5, 0.5], u=[0.0, 1.0, -1.0, 2.0, 1 - 2.0 ** -24, 0.5, 0.9, 0.99, 1.0, 0.1, 0.2, 0.3])


@pytest.mark.parametrize("p", [0.999, 0.99999, 1 - 2.0 ** -22, 1 - 2.0 ** -24])
def test_mass_close_to_all(lib, p):
    x = normal(4, 20000, 12)
    x[1] *= 5
    x[2] *= 0.1
    x[3] = np.linspace(0, -60, 20000)
    check(lib, x, "f32", t=[1.0] * 4, p=[p] * 4, u=[0.9999, 0.5, 0.99999, 0.999999])


def test_peaked_rows_with_a_long_tail(lib):
    """One token holds nearly everything; the cut lies far below it."""
    x = normal(4, 128256, 13, 1.0)
    x[:, 77] = 40.0
    check(lib, x, "f32", t=[1.0] * 4, p=[0.9, 1 - 2.0 ** -24, 1.0, 0.5], k=[0, 0, 20000, 2000], u=[0.5, 0.9999999, 0.9999999, 0.5])


@pytest.mark.parametrize("rows,vocab", [(1, 262144), (300, 700), (160, 32000), (40, 128256)])
def test_batches(lib, rows, vocab):
    rng = np.random.default_rng(rows)
    t, k = rng.choice([0.0, 0.6, 1.0, 1.3], rows), rng.choice([0, 1, 20, 500, 5000], rows)
    p, m = rng.choice([0.5, 0.9, 0.95, 1.0], rows), rng.choice([0.0, 0.01, 0.2], rows)
    check(lib, normal(rows, vocab, rows + 1), "f32", t=t, k=k, p=p, m=m, u=rng.random(rows).astype(np.float32))


@pytest.mark.parametrize("kind,shift", [("f32", 1), ("f32", 3), ("bf16", 1), ("f16", 5), ("bf16", 8)])
def test_rows_that_start_anywhere(lib, kind, shift):
    check(lib, normal(3, 1003, 14), kind, k=[20] * 3, u=[0.2, 0.6, 0.9], ld=1005, shift=shift)


def test_defaults(lib):
    rng = np.random.default_rng(15)
    check(lib, normal(8, 5000, 16), "f32", u=rng.random(8).astype(np.float32))


def test_frequencies_follow_the_weights(lib):
    """Evenly spread numbers pick each token as often as its weight says, to one number."""
    x = np.tile(np.log(np.array([1, 2, 3, 4, 6], np.float32)), (1600, 1))
    u = (np.arange(1600) + 0.5) / 1600
    got = check(lib, x, "f32", u=u)
    assert np.abs(np.bincount(got, minlength=5) - 1600 * np.array([1, 2, 3, 4, 6]) / 16).max() <= 1


def test_a_row_does_not_depend_on_its_batch_and_graphs_replay(lib):
    """The same row alone, in a batch, on another stream, and in a recording that is replayed after the numbers have changed."""
    x = torch.from_numpy(normal(64, 32000, 17)).cuda()
    u = torch.rand(64, device="cuda")
    k, p = torch.full((64,), 300, dtype=torch.int32, device="cuda"), torch.full((64,), 0.95, device="cuda")

    def run(rows, first=0, stream=None, out=None):
        out = torch.empty(rows, dtype=torch.int64, device="cuda") if out is None else out
        assert lib.bpd_sample_cuda(x.data_ptr() + first * 32000 * 4, 0, 32000, rows, 32000, None, k.data_ptr(), p.data_ptr(), None, u.data_ptr() + 4 * first, out.data_ptr(), None, stream) == 0
        return out

    torch.cuda.synchronize()
    batch = run(64)
    alone = torch.cat([run(1, i) for i in range(64)])
    torch.cuda.synchronize()
    assert torch.equal(batch, alone)
    s, out = lib.bpdq_stream_create(), torch.empty(64, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    assert lib.bpdq_graph_begin(s) == 0
    run(64, stream=s, out=out)
    g = lib.bpdq_graph_end(s)
    assert g
    for _ in range(2):
        u.copy_(torch.rand(64, device="cuda"))
        torch.cuda.synchronize()
        assert lib.bpdq_graph_launch(g, s) == 0 and lib.bpdq_stream_sync(s) == 0
        want = run(64)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    lib.bpdq_graph_destroy(g)
    lib.bpdq_stream_destroy(s)


def test_settings_that_are_no_numbers(lib):
    """NaN is no cut, and no temperature above 0; shares below 0 are the least ones."""
    nan = float("nan")
    x = np.random.default_rng(5).normal(0, 2, (6, 3000)).astype(np.float32)
    check(lib, x, "f32", t=[1, 1, nan, 0.7, 1, 1], k=[0, 50, 0, 0, 0, 0], p=[nan, nan, 0.9, 0.8, -1, 1], m=[0.01, nan, 0.1, nan, 0, -0.5], u=[0.1, 0.4, 0.6, 0.9, 0.99, 0.7])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("s", SETTINGS, ids=str)
@pytest.mark.parametrize("t", [0.0, 0.8])
def test_zeros_of_both_signs(lib, kind, s, t):
    """They are equal: the lowest index goes first, among the largest logits and at a cut with more of them than are sorted."""
    rng = np.random.default_rng(18)
    x = -np.abs(normal(6, 9000, 19)) - 0.5
    x[0, 5], x[0, 100], x[0, 8000] = -0.0, 0.0, 0.0
    x[1, [4, 7]], x[1, 2000] = 0.0, -0.0
    x[2:] = np.where(rng.random((4, 9000)) < 0.5, rng.choice(np.array([0.0, -0.0], np.float32), (4, 9000)), x[2:])
    x[3:5, ::1000] = 1.0
    x[5, :4000] = -0.0
    x[5, 4000:] = 0.0
    check(lib, x, kind, t=[t] * 6, u=[0.1, 0.5, 0.2, 0.6, 0.9, 0.7], **settings(6, s))
