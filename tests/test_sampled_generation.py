"""Requests whose tokens are sampled: the engine's part with a model that keeps count, and both kinds of models on the device, their choices against the
definition in 64 bits from the logits that the same steps give."""
import json

import numpy as np
import pytest

from bpd_substrate_b200 import _build, capi, generate, llama
from bpd_substrate_b200.engine import Engine, Request
from bpd_substrate_b200.sampling import Sampling
from bpd_substrate_b200.sequences import Sequence
from tests import hybrid_models as hm
from tests import test_hybrid_gpu as hybrid
from tests.test_hybrid_host import FakeModel
from tests.test_sample_gpu import oracle


@pytest.mark.parametrize("bad", [dict(temperature=-0.5), dict(temperature=float("inf")), dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=2 ** 31),
                                 dict(top_p=0.0), dict(top_p=1.5), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.1), dict(min_p=float("nan"))])
def test_rules_that_make_no_sense(bad):
    with pytest.raises(ValueError):
        Sampling(**bad)


class SamplingModel(FakeModel):
    """The next token is a number of the request's, so what it was given shows in what comes out."""

    def __init__(self, **kw):
        super().__init__(**kw)
        self.given = {}

    def sample(self, seq, tokens, rule, u):
        self.step(seq, tokens, [len(tokens) - 1], False)
        self.given.setdefault(rule.seed, []).append(u)
        return int(u * self.vocab) if rule.top_k != 1 else -1


@pytest.mark.parametrize("slots,portion", [(1, 4), (3, 2)])
def test_engine_hands_each_request_its_own_numbers(slots, portion):
    m = SamplingModel()
    e = Engine(m, slots, portion)
    rule = Sampling(0.7, seed=10)
    prompts = [[3, 4, 5, 6, 7], [1], [2, 2]]
    out = e.generate(prompts, 5, sampling=rule)
    for i, tokens in enumerate(out):
        u = np.random.Generator(np.random.PCG64(10 + i)).random(5, dtype=np.float32)
        assert m.given[10 + i] == [float(x) for x in u] and tokens == [int(float(x) * 50) for x in u]
    assert not e.live
    # the same request gives the same tokens, alone or beside a greedy one
    a, b = e.run([Request([1], 5, sampling=Sampling(0.7, seed=11)), Request([2], 3)])
    assert a.output == out[1] and b.output == [2, 4, 8]
    assert e.run([a.__class__([1], 5, frozenset([out[1][2]]), Sampling(0.7, seed=11))])[0].output == out[1][:out[1].index(out[1][2]) + 1]


def test_no_token_left():
    with pytest.raises(ValueError):
        Engine(SamplingModel(), 1, 4).generate([[1]], 2, sampling=Sampling(top_k=1))


def test_the_models_own_library_has_the_sampler():
    assert "sample.cu" in _build.PARTS["hybrid"]


RULES = [Sampling(0.8, seed=3), Sampling(1.3, top_k=9, seed=4), Sampling(0.9, top_p=0.7, seed=5), Sampling(2.0, top_k=30, top_p=0.9, min_p=0.2, seed=6)]


def expected(e, prompt, n, rule, seed):
    """By the definition, from the logits of the same steps."""
    numbers, out, part = np.random.Generator(np.random.PCG64(seed)), [], list(prompt)
    while len(out) < n:
        for at in range(0, len(part), e.portion):
            piece = part[at:at + e.portion]
            logits, _ = e.feed("check", piece, [len(piece) - 1])
        f = np.float32
        out.append(oracle(logits[0].astype(np.float64), float(f(rule.temperature)), rule.top_k, float(f(rule.top_p)), float(f(rule.min_p)), float(numbers.random(dtype=f)))[0])
        part = out[-1:]
    e.end("check")
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_hybrid(lib, dtype):
    cfg = hm.config(97, 64, [hm.layer("retention", hm.retention(2, 16, 16, 16, [0.5, 0.98]), 33)])
    m = hybrid.device(cfg, hm.weights(cfg, 5), lib, dtype, capacity=64)
    e = Engine(m, slots=2, portion=4)
    prompts = [hm.tokens(cfg, 11, 6), hm.tokens(cfg, 1, 7)]
    for rule in RULES:
        assert e.generate(prompts, 12, sampling=rule) == [expected(e, p, 12, rule, rule.seed + i) for i, p in enumerate(prompts)], rule
    greedy = e.generate(prompts, 12)
    assert e.generate(prompts, 12, sampling=Sampling(0.0)) == greedy == e.generate(prompts, 12, sampling=Sampling(1.0, top_k=1))
    e.close()
    m.close()


@pytest.mark.gpu
def test_llama(lib):
    cfg = llama.make_config(n_layers=2, n_heads=4, n_kv_heads=2, head_dim=32, ffn_dim=256, vocab_size=96, max_seq_len=48)
    m = llama.DeviceLlama(llama.SyntheticLlama(cfg, seed=3), lib)
    e = Engine(m, slots=2, portion=3)
    prompts = [[5, 9, 33, 2], [7]]
    for rule in RULES:
        assert e.generate(prompts, 8, sampling=rule) == [expected(e, p, 8, rule, rule.seed + i) for i, p in enumerate(prompts)], rule
    greedy = e.generate(prompts, 8)
    assert e.generate(prompts, 8, sampling=Sampling(0.0)) == greedy == e.generate(prompts, 8, sampling=Sampling(1.0, top_k=1))
    e.close()
    m.close()


@pytest.mark.gpu
def test_command(lib, tmp_path, capsys):
    cfg = hm.config(97, 64, [hm.layer("retention", hm.retention(2, 16, 16, 16, [0.5, 0.98]), 33)])
    hybrid.save_model(tmp_path, cfg, hm.weights(cfg, 5))
    args = ["--model", str(tmp_path), "--prompt", "5 17 3", "--prompt", "8", "--max-new", "6", "--capacity", "32", "--dtype", "float32"]
    said = []
    for extra in ([], ["--temperature", "0.9", "--top-k", "20", "--top-p", "0.9", "--min-p", "0.01", "--seed", "7"], ["--temperature", "0.9", "--top-k", "1"]):
        assert generate.main(args + extra) == 0
        said.append([json.loads(line)["output"] for line in capsys.readouterr().out.splitlines()])
    assert said[0] == said[2] and all(len(o) == 6 for out in said for o in out)
    m = hybrid.device(cfg, hm.weights(cfg, 5), lib, "float32", capacity=32)
    e = Engine(m, slots=2)
    assert said[1] == e.generate([[5, 17, 3], [8]], 6, sampling=Sampling(0.9, 20, 0.9, 0.01, 7))
    e.close()
    m.close()


@pytest.mark.gpu
@pytest.mark.parametrize("sampling", [None, Sampling(0.8, seed=1)])
def test_a_token_without_an_embedding_raises(lib, sampling):
    """What the device reports of a step is an error of that step, however its token is chosen."""
    cfg = llama.make_config(n_layers=1, n_heads=4, n_kv_heads=2, head_dim=32, ffn_dim=256, vocab_size=96, max_seq_len=48)
    m = llama.DeviceLlama(llama.SyntheticLlama(cfg, seed=3), lib)
    e = Engine(m, slots=1, portion=8)
    try:
        with pytest.raises(capi.BpdqError):
            e.generate([[5, 96, 7]], 2, sampling=sampling)
    finally:
        lib.bpdq_clear_status()
        e.close()
        m.close()


def test_what_the_device_reports_of_a_sampled_step_is_raised():
    """The same without a device: the library says after the step that something in it went wrong."""
    class Lib:
        status = 0

        def __getattr__(self, name):
            return lambda *args: 1 << 20 if name == "bpdq_alloc" else 0

        def bpdq_last_status(self):
            return self.status

    class Sampler:
        def pick(self, logits, vocab, rule, u):
            return 7

    m = llama.DeviceLlama.__new__(llama.DeviceLlama)
    m.lib, m.cfg, m.stream, m.vocab, m.weights, m._sampler = Lib(), llama.make_config(1, 4, 2, 32, 256, 96, 48), None, 96, capi.LlamaWeights(), Sampler()
    m._offsets = {"k": 0, "v": 0}
    seq = Sequence(0, 1 << 20, 48)
    assert m.sample(seq, [1, 2], Sampling(), 0.5) == 7 and seq.length == 2
    m.lib.status = -4
    with pytest.raises(capi.BpdqError):
        m.sample(seq, [3], Sampling(), 0.5)
    assert seq.length == 2


def test_an_engine_goes_on_after_a_request_that_fails():
    """Its slot and those of the requests beside it are free again."""
    e = Engine(SamplingModel(), 2, 4)
    for _ in range(3):
        with pytest.raises(ValueError):
            e.run([Request([1], 5), Request([2, 3], 2, sampling=Sampling(top_k=1)), Request([4], 2)])
        assert not e.live and len(e.slots.free) == 2
    assert e.generate([[1], [2], [3]], 3) == [[1, 2, 4], [2, 4, 8], [3, 6, 12]]
    # a sequence that the caller feeds by itself stays
    e.feed("mine", [5])
    with pytest.raises(ValueError):
        e.generate([[1]], 2, sampling=Sampling(top_k=1))
    assert list(e.live) == ["mine"] and e.feed("mine", [6], [0])[1].tolist() == [11]


@pytest.mark.parametrize("seed", [-1, 0.5, "one", None])
def test_seeds_that_make_no_sense(seed):
    with pytest.raises(ValueError):
        Sampling(seed=seed)


def test_a_sampled_step_without_tokens():
    m = llama.DeviceLlama.__new__(llama.DeviceLlama)
    m.lib = m.cfg = None                        # (nothing of the device is touched)
    m._sampler, m.vocab = object(), 96
    seq = Sequence(0, 1 << 20, 48)
    with pytest.raises(ValueError):
        m.sample(seq, [], Sampling(), 0.5)
