"""The operators of one step of many answers to one prompt, as cases that can be timed: attention of a batch whose texts share a long
prefix, products with weights in 8-bit floating point, and the log probabilities of the tokens that were drawn.

Every operator has its plain form here, in elementary torch operations on 32-bit floats; where `own` is true, run() calls the
package instead.  Both work on the tensors that prepare() makes; a program that uses the package holds them through the
package's handles (views of the same device memory, nothing is copied), so prepare() makes those too.

A plane of 4 bits [rows x cols] is one buffer: the codes, two to a byte (the even column in the low half), row after row; then
for each row and each group of 32 columns the f16 pair (scale, lowest).  A value is lowest + code * scale.

A tensor of 8 bits [rows x cols] is one buffer: the e4m3 codes, row after row; then the 32-bit scales, one for every 128 columns
of a row, or, for weights, one for every tile of 128 rows and 128 columns.  A value is code * scale.
"""
import math

import torch

own = False

VOCAB = 32000
GROUP = 32
BLOCK = 128
LARGEST = 448.0  # of e4m3
CACHE_BYTES = {"f16": 2.0, "f32": 4.0, "q4": 0.5 + 4.0 / GROUP}  # of a value

# heads and head size of the package's workloads; heads that share keys and values in groups are the generic shape of 8 kv heads
SHAPE_SMALL = dict(heads=16, kv=16, hd=64)
SHAPE_7B = dict(heads=32, kv=32, hd=128)
SHAPE_13B = dict(heads=40, kv=40, hd=128)
GROUPED = dict(heads=32, kv=8, hd=128)
GROUPED_WIDE = dict(heads=64, kv=8, hd=128)


def listed():
    return [
        # one token of four answers to a question of some paragraphs
        dict(name="attend-few", kind="attend", f16=True, cache="f16", **SHAPE_7B, seqs=4, n=1, prefix=383, start=20, rows=64),
        # one token of sixty-four answers to a long document, some just begun, one slot idle
        dict(name="attend-answers", kind="attend", f16=True, cache="f16", **GROUPED, seqs=64, n=1, prefix=6001, start=300, rows=512),
        # sixteen questions to a whole book, everything kept in 4 bits
        dict(name="attend-book-q4", kind="attend", f16=True, cache="q4", **GROUPED_WIDE, seqs=16, n=1, prefix=65700, start=200, rows=256),
        # two drafted tokens and the one before them, of eight answers in the default mode of 32 bits
        dict(name="attend-drafts-f32", kind="attend", f16=False, cache="f32", **SHAPE_7B, seqs=8, n=3, prefix=1031, start=77, rows=128),
        # sixteen questions of 61 tokens, read at once behind the text that they ask about
        dict(name="attend-questions", kind="attend", f16=True, cache="f16", **SHAPE_13B, seqs=16, n=61, prefix=2107, start=0, rows=64),
        # the log probabilities of the tokens just drawn for sixteen answers, with five alternatives each
        dict(name="logprobs-step", kind="logprobs", f16=False, n=16, tokens=1, top=5, temperature=0.8),
        # the log probabilities of a document's own tokens, with twenty alternatives each
        dict(name="logprobs-document", kind="logprobs", f16=True, n=2048, tokens=1, top=20, temperature=1.0),
        # one row through an attention output product
        dict(name="product-step", kind="product", source="f16", result="f16", m=1, n=4096, k=4096),
        # sixteen answers through the output head
        dict(name="product-head", kind="product", source="f16", result="f32", m=16, n=32000, k=4096),
        # sixty-four answers through the first product of a feed-forward block
        dict(name="product-answers", kind="product", source="f16", result="f16", m=64, n=11008, k=4096),
        # a few sentences through the last product of a feed-forward block, a ragged number of rows
        dict(name="product-turn", kind="product", source="f32", result="f32", m=131, n=4096, k=11008),
        # a document through the first product of a feed-forward block, converted to 8 bits once for this product and the gate's
        dict(name="product-document", kind="product", source="f8", result="f16", m=2048, n=13824, k=5120),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "logprobs", "product", "product", "product"))
    if kind == "logprobs":
        return dict(kind=kind, f16=rng.random() < 0.5, n=_log_int(rng, 1, 1000), vocab=_log_int(rng, 500, VOCAB), tokens=rng.choice((1, 1, 2, 5)), top=rng.choice((0, 1, 5, 20, 32)),
                    temperature=round(rng.uniform(0.5, 1.2), 2))
    if kind == "product":
        return dict(kind=kind, source=rng.choice(("f16", "f16", "f32", "f8")), result=rng.choice(("f16", "f32")), m=_log_int(rng, 1, 1500), n=_log_int(rng, 200, 12000),
                    k=16 * _log_int(rng, 20, 690))
    kv = rng.choice((1, 2, 4, 8, 8, 16, 32))
    heads = kv * rng.choice([g for g in (1, 1, 2, 4, 7, 8) if kv * g <= 64])
    f16 = rng.random() < 0.7
    cache = rng.choice(("q4", "f16", "f16")) if f16 else rng.choice(("q4", "f32", "f16"))
    case = dict(kind=kind, f16=f16, cache=cache, heads=heads, kv=kv, hd=rng.choice((32, 64, 128, 128, 128)), seqs=_log_int(rng, 2, 64))
    form = rng.choice(("step", "step", "draft", "question"))
    n = 1 if form == "step" else rng.randint(2, 7) if form == "draft" else _log_int(rng, 8, 600 // case["seqs"] + 9)
    position = 2 * kv * case["hd"] * CACHE_BYTES[cache]
    most = int(50e6 / position)  # positions of 50 MB
    start = 0 if form == "question" else _log_int(rng, 1, max(2, min(500, most // case["seqs"])))
    return dict(case, n=n, prefix=_log_int(rng, 16, min(3000 if form == "question" else 20000, most)), start=start, rows=start + n + rng.randint(0, 40))


# ---------------------------------------------------------------------------------------------------------------------------


def _starts(case):
    """The position of every text's first row behind the prefix: the longest first, the others ever shorter, the last of many an idle slot."""
    seqs, top = case["seqs"], case["start"]
    starts = [max(0, top - (top * 3 * b) // (4 * seqs) - 2 * b) for b in range(seqs)]
    if seqs >= 64:
        starts[-1] = -case["n"]
    return starts


_context = None


def _ctx():
    """A program's one device context."""
    global _context
    if _context is None:
        import rllama_amd

        _context = rllama_amd.Context(0)
    return _context


def _handle(t, rows=None, cols=None, kind=None):
    """The package's handle of a torch tensor's memory."""
    import rllama_amd

    types = rllama_amd.TensorDType
    dtype = {torch.float16: types.Float16, torch.float32: types.Float32, torch.int32: types.Int32}[t.dtype] if kind is None else getattr(types, kind)
    return rllama_amd.Tensor.from_device(_ctx(), t.data_ptr(), rows or t.shape[0], cols or t.shape[1], dtype)


def _pack4(x):
    """[.., cols] values -> (codes, two to a byte; (scale, lowest) of every group), as a cache of 4 bits holds them."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP).float()
    low = g.amin(-1).half()
    scale = ((g.amax(-1) - low.float()) / 15).half()
    s = scale.float().unsqueeze(-1)
    codes = torch.where(s > 0, ((g - low.float().unsqueeze(-1)) / s).round().clamp(0, 15), torch.zeros_like(g))
    codes = codes.to(torch.uint8).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    return codes[..., 0] | (codes[..., 1] << 4), torch.stack((scale, low), -1)


def _unpack4(codes, pairs):
    """The values that codes and pairs stand for, in 32 bits."""
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], codes.shape[-1] * 2 // GROUP, GROUP).float()
    v = pairs[..., 1].float().unsqueeze(-1) + c * pairs[..., 0].float().unsqueeze(-1)
    return v.reshape(*codes.shape[:-1], codes.shape[-1] * 2)


def _plane(case, gen, spread, *shape):
    """One plane [.., rows, hd] of keys or values: a tensor, or for 4 bits the buffer with its views of codes and pairs."""
    values = torch.randn(*shape, case["hd"], generator=gen, device="cuda") * spread
    if case["cache"] != "q4":
        return dict(buffer=values.half() if case["cache"] == "f16" else values)
    count = values.numel()
    buffer = torch.empty(count // 2 + count // GROUP * 4, dtype=torch.uint8, device="cuda")
    codes = buffer[: count // 2].view(*shape, case["hd"] // 2)
    pairs = buffer[count // 2:].view(torch.float16).view(*shape, case["hd"] // GROUP, 2)
    codes[:], pairs[:] = _pack4(values)
    return dict(buffer=buffer, codes=codes, pairs=pairs)


def _to_e4m3(x, rows):
    """Values [r, c] -> (codes in e4m3; their scales), a scale for every 128 columns of `rows` rows."""
    r, c = x.shape
    down, across = -(-r // rows), -(-c // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, across * BLOCK - c, 0, down * rows - r)).view(down, rows, across, BLOCK)
    top = x.abs().amax((1, 3), keepdim=True).clamp(min=LARGEST * 2.0 ** -126)
    codes = (x * (LARGEST / top)).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8).view(down * rows, across * BLOCK)[:r, :c].contiguous(), (top / LARGEST).view(down, across)


def _eight(x, rows):
    """A tensor of 8 bits: the buffer with its views of codes and scales."""
    codes, scales = _to_e4m3(x, rows)
    buffer = torch.empty(codes.numel() + scales.numel() * 4, dtype=torch.uint8, device="cuda")
    s = dict(buffer=buffer, codes=buffer[: codes.numel()].view(codes.shape), scales=buffer[codes.numel():].view(torch.float32).view(scales.shape))
    s["codes"].copy_(codes)
    s["scales"].copy_(scales)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    kind = case["kind"]
    empty = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    if kind == "logprobs":
        # logits of a model that is sure of some continuations and unsure of others, and tokens drawn from them
        n, vocab, m, top = case["n"], case.get("vocab", VOCAB), case["tokens"], case["top"]
        logits = randn(n, vocab) * (1.0 + 2.5 * torch.rand(n, 1, generator=gen, device="cuda"))
        # (the largest of logits with noise of this kind is a draw from their distribution)
        noise = -torch.rand(n, vocab, generator=gen, device="cuda").clamp(min=1e-30).log().clamp(min=1e-30).log()
        drawn = (logits + noise).sort(-1, descending=True)[1][:, :m].int().contiguous()
        s = dict(case=case, logits=logits.half() if case["f16"] else logits, tokens=drawn, logprobs=empty(n, m), entropy=empty(n, 1))
        if top:
            s.update(top_ids=empty(n, top, dtype=torch.int32), top_logprobs=empty(n, top))
        if own:
            s["handles"] = {k: _handle(s[k]) for k in ("logits", "tokens", "logprobs", "entropy", "top_ids", "top_logprobs") if k in s}
        return s
    if kind == "product":
        # activations some of whose columns stand out, as behind a norm; weights of a spread that keeps results near one
        m, n, k = (case[x] for x in ("m", "n", "k"))
        x = randn(m, k) * torch.exp(0.7 * randn(1, k))
        s = dict(case=case, weights=_eight(randn(n, k) * k ** -0.5, BLOCK), out=empty(m, n, dtype=torch.float16 if case["result"] == "f16" else torch.float32))
        s["x"] = _eight(x, 1) if case["source"] == "f8" else x.half() if case["source"] == "f16" else x
        if own:
            s["handles"] = dict(out=_handle(s["out"]), weights=_handle(s["weights"]["buffer"], n, k, "Float8Tiles"),
                                x=_handle(s["x"]["buffer"], m, k, "Float8") if case["source"] == "f8" else _handle(s["x"]))
        return s
    b, n, h, kv, hd = (case[k] for k in ("seqs", "n", "heads", "kv", "hd"))
    dtype = torch.float16 if case["f16"] else torch.float32
    starts = _starts(case)
    s = dict(case=case, starts=starts, first=torch.tensor(starts, device="cuda"))
    # queries some of whose scores stand out, as after training
    s.update(q=(randn(b * n, h * hd) * 1.5).to(dtype), out=empty(b * n, h * hd, dtype=dtype))
    for name, spread in (("k", 1.0), ("v", 0.8)):
        s["prefix_" + name] = _plane(case, gen, spread, kv, case["prefix"])
        s[name] = _plane(case, gen, spread, b, kv, case["rows"])
    if own:
        s["handles"] = {k: _handle(s[k]) for k in ("q", "out")}
        quant = dict(kind="K4BitQuantization") if case["cache"] == "q4" else {}
        s["handles"].update({k: _handle(s[k]["buffer"], kv * case["prefix"], hd, **quant) for k in ("prefix_k", "prefix_v")})
        s["handles"].update({k: _handle(s[k]["buffer"], b * kv * case["rows"], hd, **quant) for k in ("k", "v")})
    return s


# ---------------------------------------------------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)[state["case"]["kind"]](state)


def _own_attend(s):
    case, h = s["case"], s["handles"]
    h["q"].attn_shared(h["prefix_k"], h["prefix_v"], case["prefix"], h["k"], h["v"], case["heads"], case["kv"], case["rows"], s["starts"], out=h["out"])
    return s["out"]


def _own_logprobs(s):
    h = s["handles"]
    h["logits"].token_logprobs(h["tokens"], s["case"]["temperature"], logprobs=h["logprobs"], entropy=h["entropy"], top_ids=h.get("top_ids"), top_logprobs=h.get("top_logprobs"))
    return [s[k] for k in ("logprobs", "entropy", "top_ids", "top_logprobs") if k in s]


def _own_product(s):
    h = s["handles"]
    h["x"].matrix_mul_f8(h["weights"], out=h["out"])
    return s["out"]


def _rows_of(case, plane, end):
    """The first `end` rows of every head's plane, as values in 32 bits."""
    if case["cache"] == "q4":
        return _unpack4(plane["codes"][..., :end, :], plane["pairs"][..., :end, :, :])
    return plane["buffer"][..., :end, :].float()


def _plain_attend(s):
    case = s["case"]
    b, n, h, kv, hd = (case[k] for k in ("seqs", "n", "heads", "kv", "hd"))
    group = h // kv
    end = max(1, max(s["starts"]) + n)  # rows behind the longest text's end are nobody's
    pk, pv = (_rows_of(case, s["prefix_" + x], case["prefix"]) for x in "kv")
    k, v = (_rows_of(case, s[x], end) for x in "kv")
    q = s["q"].float().view(b, n, kv, group, hd) * (1 / math.sqrt(hd))
    shared = q.permute(2, 0, 1, 3, 4).reshape(kv, b * n * group, hd)
    rows = q.permute(0, 2, 1, 3, 4).reshape(b, kv, n * group, hd)
    far = torch.matmul(shared, pk.transpose(-1, -2).contiguous())
    near = torch.matmul(rows, k.transpose(-1, -2).contiguous())
    at = torch.arange(end, device="cuda")
    pos = s["first"].unsqueeze(1) + torch.arange(n, device="cuda")
    seen = (at <= pos.unsqueeze(-1)).repeat_interleave(group, 1).unsqueeze(1)
    near = torch.where(seen, near, torch.full_like(near, -math.inf))
    by_text = lambda x: x.view(kv, b, n * group, x.shape[-1]).transpose(0, 1)  # noqa: E731
    top = torch.maximum(by_text(far.amax(-1, keepdim=True)), near.amax(-1, keepdim=True))
    far = torch.exp(far - top.transpose(0, 1).reshape(kv, b * n * group, 1))
    near = torch.exp(near - top)
    total = by_text(far.sum(-1, keepdim=True)) + near.sum(-1, keepdim=True)
    out = (by_text(torch.matmul(far, pv)) + torch.matmul(near, v)) / total
    out = out.view(b, kv, n, group, hd).permute(0, 2, 1, 3, 4)
    out = torch.where((pos >= 0).view(b, n, 1, 1, 1), out, torch.zeros_like(out))
    s["out"].copy_(out.reshape(b * n, h * hd))
    return s["out"]


def _plain_logprobs(s):
    case = s["case"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    z = (x - top) * (1.0 / case["temperature"])
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log = total.log()
    s["logprobs"].copy_(z.gather(1, s["tokens"].long()) - log)
    s["entropy"].copy_(log - (e * z).sum(-1, keepdim=True) / total)
    if not case["top"]:
        return [s["logprobs"], s["entropy"]]
    ids = x.sort(dim=-1, descending=True, stable=True)[1][:, :case["top"]]
    s["top_ids"].copy_(ids)
    s["top_logprobs"].copy_(z.gather(1, ids) - log)
    return [s["logprobs"], s["entropy"], s["top_ids"], s["top_logprobs"]]


def _values(codes, scales, rows):
    """What codes and scales stand for, in 32 bits."""
    r, c = codes.shape
    scales = scales.repeat_interleave(rows, 0)[:r].repeat_interleave(BLOCK, 1)[:, :c]
    return codes.view(torch.float8_e4m3fn).float() * scales


def _plain_product(s):
    w = s["weights"]
    codes, scales = (s["x"]["codes"], s["x"]["scales"]) if s["case"]["source"] == "f8" else _to_e4m3(s["x"], 1)
    s["out"].copy_(torch.matmul(_values(codes, scales, 1), _values(w["codes"], w["scales"], BLOCK).t()))
    return s["out"]


_run_own = dict(attend=_own_attend, logprobs=_own_logprobs, product=_own_product)
_run_plain = dict(attend=_plain_attend, logprobs=_plain_logprobs, product=_plain_product)


# ---------------------------------------------------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        n, vocab = case["n"], case.get("vocab", VOCAB)
        return {"bytes": n * (vocab * (2 if case["f16"] else 4) + 4 * (2 * case["tokens"] + 1 + 2 * case["top"])), "flops": 5 * n * vocab}
    if kind == "product":
        m, n, k = (case[x] for x in ("m", "n", "k"))
        across = -(-k // BLOCK)
        x = {"f16": 2 * k, "f32": 4 * k, "f8": k + 4 * across}[case["source"]]
        return {"bytes": m * x + n * k + 4 * across * -(-n // BLOCK) + m * n * (2 if case["result"] == "f16" else 4), "flops": 2.0 * m * n * k}
    b, n, h, kv, hd = (case[k] for k in ("seqs", "n", "heads", "kv", "hd"))
    es, ec = 2 if case["f16"] else 4, CACHE_BYTES[case["cache"]]
    read, pairs = case["prefix"], 0
    for s in _starts(case):
        read += max(0, s + n)
        pairs += sum(case["prefix"] + s + i + 1 for i in range(n) if s + i >= 0)
    return {"bytes": 2 * b * n * h * hd * es + 2 * read * kv * hd * ec, "flops": 4.0 * hd * h * pairs}


# ---------------------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    return dict(attend=_exact_attend, logprobs=_exact_logprobs, product=_exact_product)[case["kind"]](prepare(case, seed))


def _exact_logprobs(s):
    top = s["case"]["top"]
    p = torch.log_softmax(s["logits"].double() / s["case"]["temperature"], -1)
    weight = p.exp()
    entropy = -(weight * p).sum(-1, keepdim=True)
    given = torch.stack([p[i, t.long()] for i, t in enumerate(s["tokens"])])
    if not top:
        return [given, entropy]
    return [given, entropy, None, p.sort(-1, descending=True)[0][:, :top]]


def _exact_product(s):
    case, w = s["case"], s["weights"]
    m, n, k = (case[x] for x in ("m", "n", "k"))
    if case["source"] == "f8":
        x = _decode(s["x"]["codes"])
        scales = s["x"]["scales"].double()
    else:
        x, scales = s["x"].double(), []
        for c in range(0, k, BLOCK):
            part = x[:, c:c + BLOCK]
            largest = part.abs().max(1, keepdim=True)[0].float()
            largest = torch.where(largest > LARGEST * 2.0 ** -126, largest, torch.full_like(largest, LARGEST * 2.0 ** -126))
            # the product of two numbers of 24 bits is exact in 64 bits, so this rounds it once to 32
            t = (part * (LARGEST / largest).double()).float().double().clamp(-LARGEST, LARGEST)
            step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
            x[:, c:c + BLOCK] = torch.round(t / step) * step
            scales.append((largest / LARGEST).double())
        scales = torch.cat(scales, 1)
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for i, c in enumerate(range(0, k, BLOCK)):
        part = x[:, c:c + BLOCK] @ _decode(w["codes"][:, c:c + BLOCK]).T
        y += part * scales[:, i:i + 1] * w["scales"].double()[:, i].repeat_interleave(BLOCK)[:n]
    return y


def _decode(codes):
    """e4m3 by its bits: a sign, four of the exponent, three behind the point."""
    c = codes.to(torch.int64)
    exponent, mantissa = (c >> 3) & 15, (c & 7).double()
    size = torch.where(exponent > 0, (8 + mantissa) * torch.exp2(exponent.double() - 10), mantissa * 2.0 ** -9)
    return torch.where(c >= 128, -size, size)


def _exact_rows(case, plane, end):
    """One head's first `end` rows in 64 bits."""
    if case["cache"] != "q4":
        return plane["buffer"][:end].double()
    codes, pairs = plane["codes"][:end], plane["pairs"][:end].double()
    x = torch.empty(end, case["hd"], dtype=torch.float64, device="cuda")
    x[:, 0::2], x[:, 1::2] = (codes % 16).double(), (codes // 16).double()
    return x * pairs[..., 0].repeat_interleave(GROUP, 1) + pairs[..., 1].repeat_interleave(GROUP, 1)


def _exact_attend(s):
    case = s["case"]
    b, n, h, kv, hd = (case[k] for k in ("seqs", "n", "heads", "kv", "hd"))
    group = h // kv
    q = s["q"].view(b, n, kv, group, hd)
    out = torch.zeros(b, n, kv, group, hd, dtype=torch.float64, device="cuda")
    part = lambda plane, *at: {k: x[at] for k, x in plane.items() if case["cache"] != "q4" or k != "buffer"}  # noqa: E731
    for j in range(kv):
        pk, pv = (_exact_rows(case, part(s["prefix_" + x], j), case["prefix"]) for x in "kv")
        for i in range(b):
            last = s["starts"][i] + n
            if last <= 0:
                continue
            k, v = (torch.cat((p, _exact_rows(case, part(s[x], i, j), last))) for x, p in (("k", pk), ("v", pv)))
            z = q[i, :, j].double().reshape(n * group, hd) @ k.T / hd ** 0.5
            at = torch.arange(last, device="cuda")
            pos = torch.arange(s["starts"][i], last, device="cuda").repeat_interleave(group)
            z[:, case["prefix"]:].masked_fill_(at > pos[:, None], -math.inf)
            y = torch.softmax(z, -1) @ v
            out[i, :, j] = torch.where((pos >= 0)[:, None], y, torch.zeros_like(y)).view(n, group, hd)
    return out.view(b * n, h * hd)
