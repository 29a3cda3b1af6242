"""The operators of a long-context speculative step, as cases that can be timed: the append of a projection's rows to the caches
(norms of queries and keys per head, position rotation, cache write), attention over caches of 16, 32 or 4 bits with a sliding
window and first tokens that stay visible, the probabilities of rows of logits, and the verification of drafted tokens.

Every operator has its plain form here, in elementary torch operations on 32-bit floats; where `own` is true, run() calls the
package instead.  Both work on the tensors that prepare() makes; a program that uses the package holds them through the
package's handles (views of the same device memory, nothing is copied), so prepare() makes those too.

A 4-bit cache plane [rows x cols] is one buffer: the codes, two to a byte (the even column in the low half), row after row; then
for each row and each group of 32 columns the f16 pair (scale, lowest).  A value is lowest + code * scale.
"""
import math

import torch

own = False

VOCAB = 32000
GROUP = 32
EPS = 1e-6

# heads and head size of the package's workloads; heads that share keys and values in groups are the generic shape of 8 kv heads
SHAPE_SMALL = dict(heads=16, kv=16, hd=64)
SHAPE_7B = dict(heads=32, kv=32, hd=128)
SHAPE_13B = dict(heads=40, kv=40, hd=128)
GROUPED = dict(heads=32, kv=8, hd=128)
GROUPED_WIDE = dict(heads=64, kv=8, hd=128)


def listed():
    return [
        # the append of one token in the middle of a chat: a launch, and little else
        dict(name="append-step", kind="append", f16=True, cache="f16", **SHAPE_7B, seqs=1, n=1, start=383, rows=512, halves=False),
        # the append of a long prompt's rows to a cache of 4 bits, behind a short text that is there already
        dict(name="append-prompt-q4", kind="append", f16=True, cache="q4", **GROUPED, seqs=1, n=1500, start=100, rows=1600, halves=True),
        # one token of a chat in the middle of its answer
        dict(name="attend-step", kind="attend", f16=True, cache="f16", **SHAPE_7B, seqs=1, n=1, start=383, rows=512, window=0, sinks=0),
        # one token behind a whole book, kept in 4 bits
        dict(name="attend-step-q4-book", kind="attend", f16=True, cache="q4", **GROUPED_WIDE, seqs=1, n=1, start=65700, rows=66000, window=0, sinks=0),
        # sixteen endless chats, one token each, every one at its own place, some shorter than the window and one slot idle
        dict(name="attend-chats-window", kind="attend", f16=True, cache="f16", **GROUPED, seqs=16, n=1, start=8000, rows=8192, window=1024, sinks=4),
        # five drafted tokens looked at together in the default mode of 32 bits
        dict(name="attend-draft-f32", kind="attend", f16=False, cache="f32", **SHAPE_7B, seqs=1, n=5, start=2107, rows=2240, window=0, sinks=0),
        # a document at the largest length the package's benchmark names
        dict(name="attend-document", kind="attend", f16=True, cache="f16", **SHAPE_13B, seqs=1, n=2048, start=0, rows=2048, window=0, sinks=0),
        # the next piece of a long text that is read through a window, from a cache of 4 bits
        dict(name="attend-piece-q4-window", kind="attend", f16=True, cache="q4", **GROUPED, seqs=1, n=1500, start=6001, rows=7600, window=1024, sinks=4),
        # the probabilities of four drafted tokens and the one behind them
        dict(name="probabilities-step", kind="probabilities", f16=False, n=5, temperature=0.8),
        # the same for a batch of 64 chats
        dict(name="probabilities-chats", kind="probabilities", f16=True, n=320, temperature=0.7),
        # the verification of four drafted tokens
        dict(name="verify-step", kind="verify", seqs=1, k=4, vocab=VOCAB),
        # the same for 64 chats and seven drafted tokens each
        dict(name="verify-chats", kind="verify", seqs=64, k=7, vocab=VOCAB),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice((1, 2, 4, 8, 8, 16, 32))
    return dict(heads=kv * rng.choice([g for g in (1, 1, 2, 4, 7, 8) if kv * g <= 64]), kv=kv, hd=rng.choice((32, 64, 128, 128, 128)))


def draw(rng):
    kind = rng.choice(("append", "append", "attend", "attend", "attend", "attend", "attend", "probabilities", "verify"))
    if kind == "probabilities":
        return dict(kind=kind, f16=rng.random() < 0.5, n=_log_int(rng, 1, 320), vocab=_log_int(rng, 500, VOCAB), temperature=round(rng.uniform(0.5, 1.2), 2))
    if kind == "verify":
        return dict(kind=kind, seqs=_log_int(rng, 1, 64), k=rng.randint(1, 7), vocab=_log_int(rng, 500, VOCAB))
    f16 = rng.random() < 0.7
    cache = rng.choice(("q4", "f16")) if f16 else rng.choice(("q4", "f32", "f16"))
    case = dict(kind=kind, f16=f16, cache=cache, **_heads(rng))
    if kind == "append":
        seqs = rng.choice((1, 1, 1, 4, 16))
        n, start = _log_int(rng, 1, 1500 // seqs), _log_int(rng, 1, 1000)
        return dict(case, seqs=seqs, n=n, start=start, rows=start + n + rng.randint(0, 100), halves=rng.random() < 0.5)
    case.update(window=0, sinks=0)
    if rng.random() < 0.4:
        case.update(window=_log_int(rng, 16, 2048), sinks=rng.choice((0, 1, 4, 16)))
    form = rng.choice(("step", "step", "draft", "prompt"))
    if form == "prompt":
        n, seqs = _log_int(rng, 17, 1800 if f16 else 300), 1
        start = 0 if rng.random() < 0.5 else _log_int(rng, 1, 2000)
    else:
        n = 1 if form == "step" else rng.randint(2, 9)
        seqs = rng.choice((1, 1, 3, 16))
        start = _log_int(rng, 1, 40000 // seqs)
    return dict(case, seqs=seqs, n=n, start=start, rows=start + n + rng.randint(0, 100))


# ---------------------------------------------------------------------------------------------------------------------------


def _starts(case):
    """The position of every sequence's first row: the longest first, the others ever shorter, the last of many an idle slot."""
    seqs, top = case["seqs"], case["start"]
    starts = [max(0, top - (top * 3 * b) // (4 * seqs) - 7 * b) for b in range(seqs)]
    if case["kind"] == "attend" and seqs >= 16:
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


def _handle(t, rows=None, cols=None, q4=False):
    """The package's handle of a torch tensor's memory."""
    import rllama_amd

    kind = rllama_amd.TensorDType
    dtype = kind.K4BitQuantization if q4 else {torch.float16: kind.Float16, torch.float32: kind.Float32, torch.int32: kind.Int32}[t.dtype]
    return rllama_amd.Tensor.from_device(_ctx(), t.data_ptr(), rows or t.shape[0], cols or t.shape[1], dtype)


def _pack(x):
    """[.., cols] values -> (codes, two to a byte; (scale, lowest) of every group), as the cache of 4 bits holds them."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP).float()
    low = g.amin(-1).half()
    scale = ((g.amax(-1) - low.float()) / 15).half()
    broken = ~(g.isfinite().all(-1) & low.isfinite() & scale.isfinite())
    low = torch.where(broken, torch.full_like(low, float("nan")), low)
    scale = torch.where(broken, torch.zeros_like(scale), scale)
    s = scale.float().unsqueeze(-1)
    codes = torch.where(s > 0, ((g - low.float().unsqueeze(-1)) / s).round().clamp(0, 15), torch.zeros_like(g))
    codes = torch.nan_to_num(codes).to(torch.uint8).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    return codes[..., 0] | (codes[..., 1] << 4), torch.stack((scale, low), -1)


def _unpack(codes, pairs):
    """The values that codes and pairs stand for, in 32 bits."""
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], codes.shape[-1] * 2 // GROUP, GROUP).float()
    v = pairs[..., 1].float().unsqueeze(-1) + c * pairs[..., 0].float().unsqueeze(-1)
    return v.reshape(*codes.shape[:-1], codes.shape[-1] * 2)


def _plane(case, gen, spread):
    """One cache plane [seqs, kv, rows, hd]: a tensor, or for 4 bits the buffer with its views of codes and pairs."""
    b, kv, rows, hd = case["seqs"], case["kv"], case["rows"], case["hd"]
    values = torch.randn(b, kv, rows, hd, generator=gen, device="cuda") * spread
    if case["cache"] != "q4":
        return dict(buffer=values.half() if case["cache"] == "f16" else values)
    count = b * kv * rows * hd
    buffer = torch.empty(count // 2 + count // GROUP * 4, dtype=torch.uint8, device="cuda")
    codes = buffer[: count // 2].view(b, kv, rows, hd // 2)
    pairs = buffer[count // 2:].view(torch.float16).view(b, kv, rows, hd // GROUP, 2)
    codes[:], pairs[:] = _pack(values)
    return dict(buffer=buffer, codes=codes, pairs=pairs)


def _plane_handle(case, plane):
    return _handle(plane["buffer"], case["seqs"] * case["kv"] * case["rows"], case["hd"], case["cache"] == "q4")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    kind = case["kind"]
    if kind == "probabilities":
        # logits of a model that is sure of some continuations and unsure of others
        n, vocab = case["n"], case.get("vocab", VOCAB)
        logits = randn(n, vocab) * (1.0 + 2.5 * torch.rand(n, 1, generator=gen, device="cuda"))
        s = dict(case=case, logits=logits.half() if case["f16"] else logits, out=torch.empty(n, vocab, device="cuda"))
        if own:
            s["handles"] = {k: _handle(s[k]) for k in ("logits", "out")}
        return s
    if kind == "verify":
        # a draft that mostly agrees with the target: its logits are the target's with some noise
        b, k, vocab = case["seqs"], case["k"], case["vocab"]
        logits = randn(b, k + 1, vocab) * 3.0
        target = logits.softmax(-1)
        draft = (logits[:, :k] + randn(b, k, vocab) * 0.7).softmax(-1)
        drafted = torch.multinomial(draft.view(b * k, vocab), 1, generator=gen).view(b, k).int()
        s = dict(case=case, target=target.view(b * (k + 1), vocab), draft=draft.view(b * k, vocab).contiguous(), drafted=drafted,
                 uniforms=torch.rand(b, k + 1, generator=gen, device="cuda"), out=torch.empty(b, k + 2, dtype=torch.int32, device="cuda"))
        if own:
            s["handles"] = {k: _handle(s[k]) for k in ("target", "draft", "drafted", "uniforms", "out")}
        return s
    b, n, h, kv, hd = (case[k] for k in ("seqs", "n", "heads", "kv", "hd"))
    dtype = torch.float16 if case["f16"] else torch.float32
    starts = _starts(case)
    s = dict(case=case, starts=starts, first=torch.tensor(starts, device="cuda"))
    if kind == "append":
        s.update(qkv=(randn(b * n, (h + 2 * kv) * hd) * 1.5).to(dtype), q=torch.empty(b * n, h * hd, dtype=dtype, device="cuda"),
                 q_norm=1 + 0.2 * randn(1, hd), k_norm=1 + 0.2 * randn(1, hd), k=_plane(case, gen, 1.0), v=_plane(case, gen, 1.0))
        # (cos, sin) of every position, in 64 bits and then rounded
        at = torch.arange(case["rows"], dtype=torch.float64, device="cuda").unsqueeze(1)
        angle = at * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
        s["freqs"] = torch.stack((angle.cos(), angle.sin()), -1).view(case["rows"], hd).float()
        s["position"] = (s["first"].unsqueeze(1) + torch.arange(n, device="cuda")).view(-1)
        s["sequence"] = torch.arange(b, device="cuda").repeat_interleave(n)
        if case["cache"] == "q4":
            for name in ("k", "v"):
                s[name]["values"] = torch.empty(b * kv * case["rows"], hd, dtype=torch.float16, device="cuda")
        if own:
            s["handles"] = {k: _handle(s[k]) for k in ("qkv", "q", "q_norm", "k_norm", "freqs")}
            s["handles"].update({k: _plane_handle(case, s[k]) for k in ("k", "v")})
            if case["cache"] == "q4":
                s["handles"].update({k + "_values": _handle(s[k]["values"]) for k in ("k", "v")})
        return s
    # queries some of whose scores stand out, as after training
    s.update(q=(randn(b * n, h * hd) * 1.5).to(dtype), out=torch.empty(b * n, h * hd, dtype=dtype, device="cuda"), k=_plane(case, gen, 1.0), v=_plane(case, gen, 0.8))
    if own:
        s["handles"] = {k: _handle(s[k]) for k in ("q", "out")}
        s["handles"].update({k: _plane_handle(case, s[k]) for k in ("k", "v")})
    return s


# ---------------------------------------------------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)[state["case"]["kind"]](state)


def _own_append(s):
    case, h = s["case"], s["handles"]
    h["qkv"].qkv_append(h["q"], h["k"], h["v"], h["freqs"], case["heads"], case["kv"], case["rows"], s["starts"], q_norm=h["q_norm"], k_norm=h["k_norm"], eps=EPS,
                        halves=case["halves"])
    if case["cache"] == "q4":
        h["k"].convert(out=h["k_values"])
        h["v"].convert(out=h["v_values"])
    return _appended(s)


def _own_attend(s):
    case, h = s["case"], s["handles"]
    h["q"].attn_window(h["k"], h["v"], case["heads"], case["kv"], case["rows"], s["starts"], window=case["window"], sinks=case["sinks"], out=h["out"])
    return s["out"]


def _own_probabilities(s):
    s["handles"]["logits"].softmax_rows(s["case"]["temperature"], out=s["handles"]["out"])
    return s["out"]


def _own_verify(s):
    h = s["handles"]
    h["drafted"].verify_draft(h["target"], h["draft"], h["uniforms"], out=h["out"])
    return s["out"]


def _appended(s):
    """The queries and what the caches hold afterwards: the whole planes of 4 bits as values, of the others the rows from the shortest text's end on."""
    if s["case"]["cache"] == "q4":
        return s["q"], s["k"]["values"], s["v"]["values"]
    first, end = min(s["starts"]), max(s["starts"]) + s["case"]["n"]
    return s["q"], s["k"]["buffer"][:, :, first:end], s["v"]["buffer"][:, :, first:end]


def _plain_append(s):
    case = s["case"]
    b, n, h, kv, hd = (case[k] for k in ("seqs", "n", "heads", "kv", "hd"))
    x = s["qkv"].float().view(b * n, h + 2 * kv, hd)
    q, k, v = x[:, :h], x[:, h:h + kv], x[:, h + kv:]
    q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
    k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    turn = s["freqs"][s["position"]].view(b * n, 1, hd // 2, 2)
    s["q"].copy_(_rotate(q, turn, case["halves"]).reshape(b * n, h * hd))
    k = _rotate(k, turn, case["halves"])
    for plane, x in ((s["k"], k), (s["v"], v)):
        if case["cache"] == "q4":
            codes, pairs = _pack(x)
            plane["codes"][s["sequence"], :, s["position"]] = codes
            plane["pairs"][s["sequence"], :, s["position"]] = pairs
            plane["values"].copy_(_unpack(plane["codes"], plane["pairs"]).view(-1, hd))
        else:
            plane["buffer"][s["sequence"], :, s["position"]] = x.to(plane["buffer"].dtype)
    return _appended(s)


def _rotate(x, turn, halves):
    cos, sin = turn[..., 0], turn[..., 1]
    if halves:
        re, im = x.chunk(2, -1)
        return torch.cat((re * cos - im * sin, re * sin + im * cos), -1)
    re, im = x[..., 0::2], x[..., 1::2]
    return torch.stack((re * cos - im * sin, re * sin + im * cos), -1).flatten(-2)


def _plain_attend(s):
    case = s["case"]
    b, n, h, kv, hd = (case[k] for k in ("seqs", "n", "heads", "kv", "hd"))
    end = max(s["starts"]) + n  # rows behind the longest text's end are nobody's
    if case["cache"] == "q4":
        k, v = (_unpack(p["codes"][:, :, :end], p["pairs"][:, :, :end]) for p in (s["k"], s["v"]))
    else:
        k, v = (p["buffer"][:, :, :end].float() for p in (s["k"], s["v"]))
    q = s["q"].float().view(b, n, kv, h // kv, hd).permute(0, 2, 1, 3, 4).reshape(b, kv, n * (h // kv), hd)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1 / math.sqrt(hd))
    at = torch.arange(end, device="cuda")
    pos = (s["first"].unsqueeze(1) + torch.arange(n, device="cuda")).unsqueeze(-1)  # [b, n, 1]
    seen = at <= pos
    if case["window"]:
        seen &= (at > pos - case["window"]) | (at < case["sinks"])
    seen = seen.repeat_interleave(h // kv, 1).unsqueeze(1)
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top.isfinite(), top, torch.zeros_like(top)))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v) / torch.where(total > 0, total, torch.ones_like(total))
    s["out"].copy_(out.view(b, kv, n, h // kv, hd).permute(0, 2, 1, 3, 4).reshape(b * n, h * hd))
    return s["out"]


def _plain_probabilities(s):
    x = s["logits"].float() * (1.0 / s["case"]["temperature"])
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return torch.div(x, x.sum(-1, keepdim=True), out=s["out"])


UNIT = 2.0 ** 31  # the draw adds up probabilities in whole numbers of this part of one


def _plain_verify(s):
    b, k, vocab = (s["case"][x] for x in ("seqs", "k", "vocab"))
    p, q = s["target"].view(b, k + 1, vocab), s["draft"].view(b, k, vocab)
    ids = s["drafted"].long().unsqueeze(-1)
    taken = s["uniforms"][:, :k] * q.gather(2, ids).squeeze(-1) < p[:, :k].gather(2, ids).squeeze(-1)
    count = taken.int().cumprod(1).sum(1)  # the drafted tokens in front of the first refusal
    row = torch.arange(b, device=p.device)
    rest = p[row, count]
    refused = (count < k).unsqueeze(1)
    rest = torch.where(refused, rest - q[row, count.clamp(max=k - 1)], rest).clamp(min=0, max=1)
    weight = (rest * UNIT).round().long()
    part = (s["uniforms"][:, k] * 2.0 ** 24).long().clamp(0, 2 ** 24 - 1)
    total = weight.sum(1)
    at = (total >> 24) * part + (((total & (2 ** 24 - 1)) * part) >> 24)
    pick = (weight.cumsum(1) <= at.unsqueeze(1)).sum(1)
    place = torch.arange(k + 1, device=p.device)
    tokens = torch.cat((s["drafted"], s["drafted"][:, :1]), 1)
    tokens = torch.where(place < count.unsqueeze(1), tokens, torch.full_like(tokens, -1))
    tokens = torch.where(place == count.unsqueeze(1), pick.int().unsqueeze(1), tokens)
    s["out"][:, 0] = count
    s["out"][:, 1:] = tokens
    return s["out"]


_run_own = dict(append=_own_append, attend=_own_attend, probabilities=_own_probabilities, verify=_own_verify)
_run_plain = dict(append=_plain_append, attend=_plain_attend, probabilities=_plain_probabilities, verify=_plain_verify)


# ---------------------------------------------------------------------------------------------------------------------------


CACHE_BYTES = {"f16": 2.0, "f32": 4.0, "q4": 0.5 + 4.0 / GROUP}


def _seen(case, p):
    """How many positions a row at position p looks at."""
    if p < 0:
        return 0
    if not case["window"]:
        return p + 1
    low = max(0, p - case["window"] + 1)
    return p + 1 - low + min(case["sinks"], low)


def work(case):
    kind = case["kind"]
    if kind == "probabilities":
        count = case["n"] * case.get("vocab", VOCAB)
        return {"bytes": count * ((2 if case["f16"] else 4) + 4), "flops": 4 * count}
    if kind == "verify":
        b, k, vocab = case["seqs"], case["k"], case["vocab"]
        return {"bytes": b * (2 * 4 * vocab + 4 * (5 * k + 3)), "flops": b * 3 * vocab}
    b, n, h, kv, hd = (case[k] for k in ("seqs", "n", "heads", "kv", "hd"))
    es, ec, starts = 2 if case["f16"] else 4, CACHE_BYTES[case["cache"]], _starts(case)
    if kind == "append":
        rows = b * n
        planes = 2 * rows * kv * hd * ec
        if case["cache"] == "q4":
            planes += 2 * b * kv * case["rows"] * hd * (ec + 2)  # the planes that are read back
        return {"bytes": rows * ((2 * h + 2 * kv) * hd * es + 4 * hd) + planes, "flops": rows * (h + kv) * hd * 7}
    read = pairs = 0
    for s in starts:
        if s + n <= 0:
            continue
        first = max(0, s)
        # the union of what the rows look at: the last row's span grown by the rows in front of it, and the first tokens
        low = max(0, first - case["window"] + 1) if case["window"] else 0
        read += s + n - low + min(case["sinks"], low)
        pairs += sum(_seen(case, s + i) for i in range(n))
    return {"bytes": 2 * b * n * h * hd * es + 2 * read * kv * hd * ec, "flops": 4.0 * hd * h * pairs}


def exact(case, seed):
    kind = case["kind"]
    if kind == "verify":
        return None  # whole numbers
    s = prepare(case, seed)
    if kind == "probabilities":
        return torch.softmax(s["logits"].double() / case["temperature"], -1)
    b, n, h, kv, hd = (case[k] for k in ("seqs", "n", "heads", "kv", "hd"))
    if kind == "append":
        return _exact_append(case, s)
    out = torch.zeros(b, n, h, hd, dtype=torch.float64, device="cuda")
    for i in range(b):
        last = s["starts"][i] + n
        if last <= 0:
            continue
        at = torch.arange(last, device="cuda")
        pos = torch.arange(s["starts"][i], last, device="cuda")[:, None]
        hidden = at > pos
        if case["window"]:
            hidden = hidden | ((at <= pos - case["window"]) & (at >= case["sinks"]))
        for j in range(h):
            k, v = (_exact_rows(case, s[p], i, j // (h // kv), last) for p in ("k", "v"))
            q = s["q"].view(b, n, h, hd)[i, :, j].double()
            z = (q @ k.T / hd ** 0.5).masked_fill(hidden, -math.inf)
            out[i, :, j] = torch.softmax(z, -1) @ v
    return torch.nan_to_num(out).view(b * n, h * hd)


def _exact_rows(case, plane, i, j, last):
    if case["cache"] != "q4":
        return plane["buffer"][i, j, :last].double()
    codes, pairs = plane["codes"][i, j, :last], plane["pairs"][i, j, :last].double()
    x = torch.empty(last, case["hd"], dtype=torch.float64, device="cuda")
    x[:, 0::2], x[:, 1::2] = (codes % 16).double(), (codes // 16).double()
    return x * pairs[..., 0].repeat_interleave(GROUP, 1) + pairs[..., 1].repeat_interleave(GROUP, 1)


def _exact_append(case, s):
    b, n, h, kv, hd = (case[k] for k in ("seqs", "n", "heads", "kv", "hd"))
    x = s["qkv"].double().view(b, n, h + 2 * kv, hd)
    half = hd // 2
    pos = torch.stack([torch.arange(a, a + n, device="cuda") for a in s["starts"]])
    re, im = s["freqs"].double()[pos].view(b, n, half, 2).unbind(-1)
    turn = torch.complex(re, im).unsqueeze(2)

    def turned(y, weight):
        y = y / (y.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * weight.double()
        y = y.unflatten(-1, (2, half)).transpose(-1, -2) if case["halves"] else y.unflatten(-1, (half, 2))
        y = torch.view_as_real(torch.view_as_complex(y.contiguous()) * turn)
        return (y.transpose(-1, -2) if case["halves"] else y).flatten(-2)

    q = turned(x[:, :, :h], s["q_norm"]).view(b * n, h * hd)
    if case["cache"] == "q4":
        return q, None, None  # a code next to its neighbour's is as good
    planes = []
    for name, y in (("k", turned(x[:, :, h:h + kv], s["k_norm"])), ("v", x[:, :, h + kv:])):
        whole = s[name]["buffer"].double()
        for i in range(b):
            whole[i, :, s["starts"][i]:s["starts"][i] + n] = y[i].transpose(0, 1)
        planes.append(whole[:, :, min(s["starts"]):max(s["starts"]) + n])
    return q, planes[0], planes[1]
