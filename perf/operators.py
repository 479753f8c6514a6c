"""The operators of serving many sequences at once, as a user calls them, beside their plain form in elementary torch operations.

op             entry point                       what it computes
append         bpd_paged_append_cuda             queries and keys of new tokens turned by their positions, keys and values put into the pages of
                                                 their sequences
attention      bpd_paged_attention_cuda          attention of new tokens over the pages of their sequences (one token each, prompts in portions, or
                                                 both in one batch), sequences that share their first pages among them
sample         bpd_sample_cuda                   a token per row of logits by temperature, top-k, top-p and min-p from given random numbers

Shapes are those of the decoders in cases.py: Llama-3-8B's heads (32 on 8 of 128, fp32 activations on an fp16 cache, or all bf16), 16 on 4 of
64, and vocabularies of 32000 and 128256.  A pool's pages are dealt to sequences in random order, as they are after a while of serving.
"""
import ctypes as C
import math
import random

import torch

own = False

TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}


def listed():
    llama = {"heads": 32, "kv_heads": 8, "dim": 128}
    small = {"heads": 16, "kv_heads": 4, "dim": 64}
    return [
        # a decode step of a small batch: latency
        {"name": "append_16x1", "op": "append", **llama, "act": "f32", "kv": "f16", "page": 16, "batch": 16, "new": 1, "context": 4000, "rot": 128, "pairs": "neighbours"},
        # a large batch of short replies, half of a head's dimensions turned
        {"name": "append_200x1", "op": "append", **small, "act": "f16", "kv": "f16", "page": 32, "batch": 200, "new": 1, "context": 1000, "rot": 32, "pairs": "halves"},
        # five prompts in one step
        {"name": "append_5x2000", "op": "append", **llama, "act": "bf16", "kv": "bf16", "page": 16, "batch": 5, "new": 2000, "context": 100, "rot": 128, "pairs": "halves"},
        # one user, late in a conversation: latency
        {"name": "decode_1x4000", "op": "attention", **llama, "act": "f32", "kv": "f16", "page": 16, "batch": 1, "new": 1, "context": 4000, "prefix": 0, "groups": 0, "cap": 0.0},
        # a batch of conversations of very different lengths
        {"name": "decode_64x8000", "op": "attention", **llama, "act": "bf16", "kv": "bf16", "page": 16, "batch": 64, "new": 1, "context": 8000, "prefix": 0, "groups": 0, "cap": 0.0},
        # portions of three prompts
        {"name": "prefill_3x2000", "op": "attention", **llama, "act": "bf16", "kv": "bf16", "page": 16, "batch": 3, "new": 2000, "context": 2000, "prefix": 0, "groups": 0, "cap": 0.0},
        # one prompt's portion among sequences that decode, the Llama's types
        {"name": "mixed_31x1000", "op": "attention", **llama, "act": "f32", "kv": "f16", "page": 16, "batch": 31, "new": 1000, "one_prompt": True, "context": 3000, "prefix": 0,
         "groups": 0, "cap": 0.0},
        # samples of one long prompt: the prefix is read once for all
        {"name": "shared_64x16000", "op": "attention", **llama, "act": "bf16", "kv": "bf16", "page": 16, "batch": 64, "new": 1, "context": 500, "prefix": 16000, "groups": 1, "cap": 0.0},
        # three instructions, each shared by several sequences, capped scores
        {"name": "shared_40x2000", "op": "attention", **small, "act": "f16", "kv": "f16", "page": 32, "batch": 40, "new": 1, "context": 300, "prefix": 2000, "groups": 3, "cap": 30.0},
        # one row, the usual cuts: latency
        {"name": "sample_1x32000", "op": "sample", "rows": 1, "vocab": 32000, "type": "f32", "top_k": True, "top_p": True, "min_p": False},
        # a batch whose rows have settings of their own, greedy ones among them
        {"name": "sample_64x128256", "op": "sample", "rows": 64, "vocab": 128256, "type": "f32", "top_k": True, "top_p": True, "min_p": True},
        # rollouts: many rows, most of the mass kept, logits of a bf16 head (many equal values)
        {"name": "sample_300x32000", "op": "sample", "rows": 300, "vocab": 32000, "type": "bf16", "top_k": False, "top_p": True, "min_p": False},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "sample"])
    if op == "sample":
        vocab = _spread(rng, 1000, 128256)
        return {"op": op, "rows": _spread(rng, 1, min(300, 64 * 128256 // vocab)), "vocab": vocab, "type": rng.choice(["f32", "f32", "f16", "bf16"]), "top_k": rng.random() < 0.6,
                "top_p": rng.random() < 0.7, "min_p": rng.random() < 0.4}
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 128), (32, 32, 64), (16, 4, 64), (8, 1, 128), (14, 2, 64), (12, 4, 96), (16, 8, 80)])
    act, kv = rng.choice([("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16")])
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "act": act, "kv": kv, "page": rng.choice([8, 16, 16, 32, 64, 128])}
    if op == "append":
        batch = _spread(rng, 1, 200)
        one = rng.random() < 0.5
        return {**case, "batch": batch, "new": 1 if one else _spread(rng, 2, max(2, 10000 // batch)), "context": _spread(rng, 1, 8000 if batch <= 16 else 1000),
                "rot": rng.choice([dim, dim, dim // 2, 0]), "pairs": rng.choice(["neighbours", "halves"])}
    kind, cap = rng.choice(["decode", "decode", "prefill", "mixed", "shared", "shared"]), rng.choice([0.0, 0.0, 0.0, 30.0])
    if kind in ("prefill", "mixed"):
        batch = _spread(rng, 1, 5) if kind == "prefill" else _spread(rng, 2, 40)
        return {**case, "batch": batch, "new": _spread(rng, 2, 2000 if kind == "prefill" and act != "f32" else 1000), "one_prompt": kind == "mixed", "context": _spread(rng, 1, 2000),
                "prefix": 0, "groups": 0, "cap": cap}
    batch = _spread(rng, 1 if kind == "decode" else 2, 128)
    if kind == "decode":
        return {**case, "batch": batch, "new": 1, "context": _spread(rng, 1, min(16000, 400000 // batch)), "prefix": 0, "groups": 0, "cap": cap}
    groups = rng.randint(1, min(4, batch))
    return {**case, "batch": batch, "new": 1, "context": _spread(rng, 1, 500), "prefix": _spread(rng, 2 * case["page"], 16000 // groups), "groups": groups, "cap": cap}


# ---- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _plan(case):
    """Lengths of a batch: (tokens that each sequence holds ahead of the call, new tokens of each, bounds of the groups, whole pages that each
    group shares).  Sequences of one prompt share its whole pages; what is left of the prompt is their own."""
    rng = random.Random(case["batch"] * 100003 + case["context"] * 101 + case["new"])
    held = [_spread(rng, max(1, case["context"] // 8), case["context"]) for _ in range(case["batch"])]
    new = [1 if case["new"] == 1 or (case.get("one_prompt") and b != case["batch"] // 2) else _spread(rng, max(1, case["new"] // 2), case["new"]) for b in range(case["batch"])]
    if case["batch"] == 1:
        held, new = [case["context"]], [case["new"]]
    n = case.get("groups", 0)
    bounds = [case["batch"] * i // n for i in range(n + 1)] if n else []
    pages = []
    for i in range(n):
        prefix = case["prefix"] - i * (case["prefix"] // 8)
        pages.append(prefix // case["page"])
        for b in range(bounds[i], bounds[i + 1]):
            held[b] += prefix
    return held, new, bounds, pages


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_paged(case, seed):
    g, page = _gen(seed), case["page"]
    act, kv = TYPES[case["act"]][0], TYPES[case["kv"]][0]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    held, new, bounds, shared = _plan(case)
    need = [-(-(h + n) // page) for h, n in zip(held, new)]
    first = {b: i for i in range(len(shared)) for b in range(bounds[i], bounds[i + 1])}      # the group of a sequence
    total = sum(need) - sum(shared[i] * (bounds[i + 1] - bounds[i] - 1) for i in range(len(shared)))
    n_pages = total + 8                                        # some pages of the pool belong to nobody
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32).cpu()
    table, at, prefix = torch.zeros(len(held), max(need), dtype=torch.int32), 0, {}
    for b, count in enumerate(need):
        i = first.get(b)
        if i is not None and i not in prefix:
            prefix[i] = order[at:at + shared[i]]
            at += shared[i]
        k = 0 if i is None else shared[i]
        if k:
            table[b, :k] = prefix[i]
        table[b, k:count] = order[at:at + count - k]
        at += count - k
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    tokens = starts[-1]
    s = {"case": case, "tokens": tokens, "new": new, "held": held,
         "k_pool": _normal(g, n_pages, kv_heads, page, dim, dtype=kv), "v_pool": _normal(g, n_pages, kv_heads, page, dim, dtype=kv),
         "table": table.cuda(), "length": _ints(held), "start": _ints(starts) if max(new) > 1 else None,
         # queries, keys and values of a token side by side, as one product leaves them
         "qkv": _normal(g, tokens, heads + 2 * kv_heads, dim, dtype=act)}
    s["q_out"] = torch.empty(tokens, heads, dim, device="cuda", dtype=act)
    if case["op"] == "append":
        half = case["rot"] // 2
        s["freq"] = (500000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(half, 1))).float()
    else:
        s["scale"] = 1.5 / math.sqrt(dim)
        s["bounds"], s["shared"] = (_ints(bounds), _ints(shared)) if shared else (None, None)
    if own:
        from bpd_substrate_b200 import capi
        at = torch.Tensor.data_ptr
        kv_desc = capi.PagedKv(heads=heads, kv_heads=kv_heads, dim=dim, act_type=TYPES[case["act"]][1], kv_type=TYPES[case["kv"]][1], page=page, n_pages=n_pages,
                               batch=len(held), max_pages=table.shape[1], page_stride=0, k=at(s["k_pool"]), v=at(s["v_pool"]), page_table=at(s["table"]),
                               length=at(s["length"]), seq_start=None if s["start"] is None else at(s["start"]))
        s["kv"] = kv_desc
        if case["op"] == "attention" and shared:
            s["groups"] = capi.PagedGroups(n=len(shared), start=at(s["bounds"]), pages=at(s["shared"]))
    return s


def _prepare_sample(case, seed):
    g, rows, vocab = _gen(seed), case["rows"], case["vocab"]
    rng = random.Random(seed)

    def setting(values, dtype, used=True):
        return torch.tensor([rng.choice(values) for _ in range(rows)], dtype=dtype, device="cuda") if used else None

    sharp = 1.0 + 2.5 * torch.rand(rows, 1, device="cuda", generator=g)          # flat rows and peaked ones
    s = {"case": case, "logits": (_normal(g, rows, vocab) * sharp).to(TYPES[case["type"]][0]), "u": torch.rand(rows, device="cuda", generator=g),
         "temperature": setting([0.6, 0.8, 1.0, 1.2] + [0.0] * (rows > 8), torch.float32), "top_k": setting([20, 50, 200] + [0] * (rows > 1), torch.int32, case["top_k"]),
         "top_p": setting([0.9, 0.95, 0.99], torch.float32, case["top_p"]), "min_p": setting([0.0, 0.02, 0.1], torch.float32, case["min_p"]),
         "token": torch.empty(rows, dtype=torch.int64, device="cuda"), "logprob": torch.empty(rows, device="cuda")}
    return s


def prepare(case, seed):
    return _prepare_sample(case, seed) if case["op"] == "sample" else _prepare_paged(case, seed)


# ---- one pass

def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_append(s):
    from bpd_substrate_b200 import capi
    c, ld, x, size = s["case"], s["qkv"].stride(0), s["qkv"].data_ptr(), s["qkv"].element_size() * s["case"]["dim"]
    capi.check(capi.load().bpd_paged_append_cuda(C.byref(s["kv"]), x, ld, s["q_out"].data_ptr(), s["q_out"].stride(0), x + c["heads"] * size, ld,
                                                 x + (c["heads"] + c["kv_heads"]) * size, ld, s["tokens"], c["rot"], int(c["pairs"] == "neighbours"), s["freq"].data_ptr(),
                                                 _stream()))
    return s["q_out"], s["k_pool"], s["v_pool"]


def _own_attention(s):
    from bpd_substrate_b200 import capi
    groups = C.byref(s["groups"]) if "groups" in s else None
    capi.check(capi.load().bpd_paged_attention_cuda(C.byref(s["kv"]), s["qkv"].data_ptr(), s["qkv"].stride(0), s["q_out"].data_ptr(), s["q_out"].stride(0), s["tokens"],
                                                    s["scale"], s["case"]["cap"], groups, _stream()))
    return s["q_out"]


def _own_sample(s):
    from bpd_substrate_b200 import capi
    c = s["case"]
    settings = [None if s[name] is None else s[name].data_ptr() for name in ("temperature", "top_k", "top_p", "min_p")]
    capi.check(capi.load().bpd_sample_cuda(s["logits"].data_ptr(), TYPES[c["type"]][1], c["vocab"], c["rows"], c["vocab"], *settings, s["u"].data_ptr(), s["token"].data_ptr(),
                                           s["logprob"].data_ptr(), _stream()))
    return s["token"], s["logprob"]


_own = {"append": _own_append, "attention": _own_attention, "sample": _own_sample}


def _places(s):
    """Sequence and position of every new token."""
    t = torch.arange(s["tokens"], device="cuda")
    if s["start"] is None:
        return t, s["length"].long()
    seq = torch.searchsorted(s["start"].long(), t, right=True) - 1
    return seq, s["length"].long()[seq] + t - s["start"].long()[seq]


def _plain_append(s):
    c = s["case"]
    heads, kv_heads, rot, half = c["heads"], c["kv_heads"], c["rot"], c["rot"] // 2
    seq, pos = _places(s)
    angle = pos.double()[:, None] * s["freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = s["qkv"][:, :heads + kv_heads].float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["pairs"] == "neighbours" else (x[..., :half], x[..., half:rot])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([a, b], -1).flatten(-2) if c["pairs"] == "neighbours" else torch.cat([a, b], -1)
    x = torch.cat([turned, x[..., rot:]], -1)
    page, slot = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    kind = s["k_pool"].dtype
    s["q_out"].copy_(x[:, :heads])
    s["k_pool"][page, :, slot] = x[:, heads:].to(kind)
    s["v_pool"][page, :, slot] = s["qkv"][:, heads + kv_heads:].to(kind)
    return s["q_out"], s["k_pool"], s["v_pool"]


def _plain_attention(s):
    c, at = s["case"], 0
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    for b, (held, n) in enumerate(zip(s["held"], s["new"])):
        seen = held + n
        pages = s["table"][b, :-(-seen // c["page"])].long()
        k, v = (s[name][pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :seen].float() for name in ("k_pool", "v_pool"))
        q = s["qkv"][at:at + n, :heads].float().reshape(n, kv_heads, heads // kv_heads, dim).permute(1, 2, 0, 3).reshape(kv_heads, -1, dim)
        w = q @ k.transpose(1, 2) * s["scale"]
        if c["cap"]:
            w = c["cap"] * torch.tanh(w / c["cap"])
        if n > 1:
            hidden = torch.arange(seen, device="cuda")[None] > held + torch.arange(n, device="cuda")[:, None]
            w = w.view(kv_heads, -1, n, seen).masked_fill(hidden, -math.inf).view(kv_heads, -1, seen)
        w = torch.exp(w - w.amax(-1, keepdim=True))
        o = w @ v / w.sum(-1, keepdim=True)
        s["q_out"][at:at + n] = o.view(heads, n, dim).transpose(0, 1)
        at += n
    return s["q_out"]


def _plain_sample(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    t = s["temperature"].double()[:, None]
    x, index = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    z = (x - x[:, :1]) / torch.where(t > 0, t, 1.0)
    w = torch.where(t > 0, torch.exp(z), (torch.arange(vocab, device="cuda") == 0).double())
    place = torch.arange(vocab, device="cuda")
    keep = torch.ones(rows, vocab, dtype=torch.bool, device="cuda")
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        keep &= (place < k) | (k <= 0)
    if s["top_p"] is not None:
        mass = torch.cumsum(w * keep, -1)
        p = s["top_p"].double()[:, None]
        keep &= (mass - w < p * mass[:, -1:]) | (p >= 1)
    if s["min_p"] is not None:
        keep &= w >= s["min_p"].double()[:, None]
    kept = torch.zeros_like(w).scatter_(1, index, w * keep)                # back in the order of the vocabulary
    mass = torch.cumsum(kept, -1)
    token = (mass <= s["u"].double()[:, None] * mass[:, -1:]).sum(-1)
    s["token"].copy_(token)
    s["logprob"].copy_(torch.log(kept.gather(1, token[:, None])[:, 0] / mass[:, -1]))
    return s["token"], s["logprob"]


_plain = {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}


# ---- what a pass cannot do without

def work(case):
    if case["op"] == "sample":
        size = 4 if case["type"] == "f32" else 2
        settings = 2 + sum(case[name] for name in ("top_k", "top_p", "min_p"))
        return {"bytes": case["rows"] * (case["vocab"] * size + 4 * settings + 12), "flops": 0}
    held, new, bounds, shared = _plan(case)
    heads, kv_heads, dim, a, tokens = case["heads"], case["kv_heads"], case["dim"], 4 if case["act"] == "f32" else 2, sum(new)
    if case["op"] == "append":
        return {"bytes": tokens * dim * ((2 * heads + 2 * kv_heads) * a + 2 * kv_heads * 2), "flops": 3 * tokens * (heads + kv_heads) * case["rot"]}
    rows = sum(h + n for h, n in zip(held, new)) - sum(p * case["page"] * (bounds[i + 1] - bounds[i] - 1) for i, p in enumerate(shared))
    pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new))
    return {"bytes": 2 * rows * kv_heads * dim * 2 + 2 * tokens * heads * dim * a, "flops": 4 * pairs * heads * dim}


# ---- the same results from the definitions in 64 bits

def exact(case, seed):
    s = _prepare_any(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["op"]](case, s)


def _prepare_any(case, seed):
    """The inputs alone."""
    global own
    mine, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = mine


def _exact_append(case, s):
    rot, heads, kv_heads, page = case["rot"], case["heads"], case["kv_heads"], case["page"]
    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    x = s["qkv"].double()
    pos = torch.cat([h + torch.arange(n, device="cuda") for h, n in zip(s["held"], s["new"])])
    # a pair as a complex number, turned by exp(i position frequency)
    turn = torch.polar(torch.ones(1, 1, dtype=torch.float64, device="cuda"), torch.outer(pos.double(), s["freq"].double()))[:, None]
    first = slice(0, rot, 2) if case["pairs"] == "neighbours" else slice(0, rot // 2)
    second = slice(1, rot, 2) if case["pairs"] == "neighbours" else slice(rot // 2, rot)
    z = torch.complex(x[:, :heads + kv_heads, first].contiguous(), x[:, :heads + kv_heads, second].contiguous()) * turn
    x[:, :heads + kv_heads, first] = z.real
    x[:, :heads + kv_heads, second] = z.imag
    at = 0
    for b, (h, n) in enumerate(zip(s["held"], s["new"])):
        p = pos[at:at + n]
        rows = s["table"][b].long()[p // page]
        k_pool[rows, :, p % page] = x[at:at + n, heads:heads + kv_heads]
        v_pool[rows, :, p % page] = x[at:at + n, heads + kv_heads:]
        at += n
    return x[:, :heads].contiguous(), k_pool, v_pool


def _exact_attention(case, s):
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.empty(s["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    at = 0
    for b, (held, n) in enumerate(zip(s["held"], s["new"])):
        pos = torch.arange(held + n, device="cuda")
        rows, slots = s["table"][b].long()[pos // page], pos % page
        for g in range(kv_heads):
            k, v = s["k_pool"][rows, g, slots].double(), s["v_pool"][rows, g, slots].double()
            for h in range(g * (heads // kv_heads), (g + 1) * (heads // kv_heads)):
                score = s["scale"] * torch.mm(s["qkv"][at:at + n, h].double(), k.T)
                if case["cap"]:
                    score = case["cap"] * torch.tanh(score / case["cap"])
                score = torch.where(pos[None] <= held + torch.arange(n, device="cuda")[:, None], score, -math.inf)
                out[at:at + n, h] = torch.softmax(score, -1) @ v
        at += n
    return out


def _exact_sample(case, s):
    tokens, logprobs = [], []
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        t = float(s["temperature"][r])
        if t <= 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            logprobs.append(0.0)
            continue
        p = torch.softmax(x / t, 0)
        order = torch.argsort(x, descending=True, stable=True)
        count = case["vocab"]
        if s["top_k"] is not None and int(s["top_k"][r]) > 0:
            count = min(count, int(s["top_k"][r]))
        q = p[order[:count]]
        most = count
        if s["top_p"] is not None and float(s["top_p"][r]) < 1:
            most = min(most, 1 + int((q.cumsum(0) < float(s["top_p"][r]) * q.sum()).sum()))
        if s["min_p"] is not None:
            most = min(most, int((q >= float(s["min_p"][r]) * q[0]).sum()))
        kept = order[:most].sort().values
        mass = p[kept].cumsum(0)
        i = int((mass <= float(s["u"][r]) * mass[-1]).sum())
        tokens.append(int(kept[i]))
        logprobs.append(float(torch.log(p[kept[i]] / mass[-1])))
    return torch.tensor(tokens, device="cuda"), torch.tensor(logprobs, dtype=torch.float64, device="cuda")
