"""Several chats with long texts, a small model drafting and a large one verifying.

    python examples/drafted_tokens.py [--chats 4] [--tokens 48] [--draft 4] [--window 96] [--cache q4|f16|f32] [--arithmetic f32|f16]
                                      [--temperature 0.8]

Both models are LLaMA-shaped stacks with grouped heads, normalised queries and keys and random weights, written out op by op:

    rows -> rmsnorm -> wq|wk|wv -> qkv_append (norms, rotation, cache rows) -> attn_window -> wo, add -> rmsnorm -> silu(w1) * w3 -> w2, add

The caches are rings: the first `sinks` positions stay, of the others the last `window` are seen, so memory does not grow with a chat; it may run on as far
as the table of angles goes (a row of head_dim numbers for every position).  A round takes
`draft` tokens from the small model one by one, runs the large one over all of them at once (one pass over its weights) and keeps what
verify_draft accepts plus the token it draws itself: the tokens are distributed as if the large model had drawn each of them, whatever the
small one proposes.  Positions that were appended for refused tokens are simply written again by the next round; the rows they took in the ring are
counted in its size (sinks + window + rows at once - 1), so that no position still seen is lost to them.
"""
import argparse
import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from rllama_amd import Context, Tensor, TensorDType  # noqa: E402

CACHES = {"f16": TensorDType.Float16, "f32": TensorDType.Float32, "q4": TensorDType.K4BitQuantization}


class Stack:
    """A transformer of random weights, with caches for `chats` texts.  f32: everything in f32.  f16: weights and what goes between the products in f16, norms and
    the residual stream in f32."""

    def __init__(self, ctx, seed, layers, dim, n_heads, n_kv_heads, head_dim, ffn, vocab, positions, chats, window, sinks, rows_at_once, cache, f16=False):
        rng = np.random.default_rng(seed)
        self.dtype = TensorDType.Float16 if f16 else TensorDType.Float32

        def weights(rows, cols):
            w = rng.standard_normal((rows, cols), np.float32) / np.float32(np.sqrt(cols))
            return Tensor.from_numpy(ctx, w.astype(np.float16) if f16 else w)

        def ones(cols):
            return Tensor.from_numpy(ctx, np.ones((1, cols), np.float32))

        self.ctx, self.n_heads, self.n_kv, self.hd, self.window, self.sinks = ctx, n_heads, n_kv_heads, head_dim, window, sinks
        self.ring = sinks + window + rows_at_once - 1  # what a pass of `rows_at_once` rows needs
        self.embedding = rng.standard_normal((vocab, dim), np.float32)
        self.freqs = Tensor.zeros(ctx, positions, head_dim, TensorDType.Float32).rope_table()
        self.layers = [dict(attention_norm=ones(dim), wqkv=weights((n_heads + 2 * n_kv_heads) * head_dim, dim), q_norm=ones(head_dim), k_norm=ones(head_dim),
                            wo=weights(dim, n_heads * head_dim), ffn_norm=ones(dim), w1=weights(ffn, dim), w3=weights(ffn, dim), w2=weights(dim, ffn),
                            k=Tensor.zeros(ctx, chats * n_kv_heads * self.ring, head_dim, cache), v=Tensor.zeros(ctx, chats * n_kv_heads * self.ring, head_dim, cache))
                       for _ in range(layers)]
        self.norm, self.output = ones(dim), weights(vocab, dim)

    def forward(self, tokens, start_pos):
        """Logits [chats * n x vocab] of tokens [chats x n], chat b's at positions start_pos[b] on (negative: padding)."""
        rows, f16 = tokens.size, self.dtype == TensorDType.Float16
        norm = lambda x, w: x.rmsnorm(w, 1e-6).convert(self.dtype) if f16 else x.rmsnorm(w, 1e-6)  # noqa: E731
        add = lambda x, y: x.add(y.convert(TensorDType.Float32) if f16 else y)  # noqa: E731
        x = Tensor.from_numpy(self.ctx, self.embedding[np.maximum(tokens, 0).reshape(-1)])
        for w in self.layers:
            qkv = norm(x, w["attention_norm"]).matrix_mul_transposed(w["wqkv"])
            q = Tensor.zeros(self.ctx, rows, self.n_heads * self.hd, self.dtype)
            qkv.qkv_append(q, w["k"], w["v"], self.freqs, self.n_heads, self.n_kv, self.ring, start_pos, q_norm=w["q_norm"], k_norm=w["k_norm"], sinks=self.sinks)
            seen = q.attn_window(w["k"], w["v"], self.n_heads, self.n_kv, self.ring, start_pos, window=self.window, sinks=self.sinks)
            x = add(x, seen.matrix_mul_transposed(w["wo"]))
            h = norm(x, w["ffn_norm"])
            x = add(x, h.matrix_mul_transposed(w["w1"]).silu_mul(h.matrix_mul_transposed(w["w3"])).matrix_mul_transposed(w["w2"]))
        return norm(x, self.norm).matrix_mul_transposed(self.output)

    def read(self, texts, rows_at_once):
        """The texts but for their last tokens into the caches, `rows_at_once` rows of each at a time, shorter texts padded on the left."""
        longest = max(len(t) for t in texts) - 1
        for first in range(-(-longest // rows_at_once) * -rows_at_once, 0, rows_at_once):
            start = [len(t) - 1 + first for t in texts]
            self.forward(np.array([[t[s + i] if s + i >= 0 else -1 for i in range(rows_at_once)] for t, s in zip(texts, start)]), start)


def draw(probs, uniforms):
    """One token per row of probabilities."""
    sums = np.cumsum(probs.astype(np.float64), 1)
    return np.minimum((sums <= uniforms[:, None] * sums[:, -1:]).sum(1), probs.shape[1] - 1).astype(np.int32)


def generate(ctx, large, small, texts, n_tokens, k, temperature, seed, rows_at_once):
    """Continues every text by at least n_tokens tokens; returns (texts, rounds, drafted tokens accepted)."""
    rng = np.random.default_rng(seed)
    texts = [list(t) for t in texts]
    goal = [len(t) + n_tokens for t in texts]
    for model in (large, small):
        model.read(texts, rows_at_once)
    chats, vocab, rounds, accepted = len(texts), large.embedding.shape[0], 0, 0
    while any(len(t) < g for t, g in zip(texts, goal)):
        pos = [len(t) - 1 for t in texts]  # of the last token, which no cache holds yet
        tokens = np.zeros((chats, k + 1), np.int32)
        tokens[:, 0] = [t[-1] for t in texts]
        draft = np.zeros((chats, k, vocab), np.float32)
        for i in range(k + 1):  # (the last pass is for the small model's caches only)
            logits = small.forward(tokens[:, i:i + 1], [p + i for p in pos])
            if i < k:
                draft[:, i] = logits.softmax_rows(temperature).to_numpy()
                tokens[:, i + 1] = draw(draft[:, i], rng.random(chats))
        target = large.forward(tokens, pos).softmax_rows(temperature)
        uniforms = Tensor.from_numpy(ctx, rng.random((chats, k + 1), np.float32))
        out = Tensor.from_numpy(ctx, tokens[:, 1:]).verify_draft(target, Tensor.from_numpy(ctx, draft.reshape(chats * k, vocab)), uniforms).to_numpy()
        for t, row in zip(texts, out):
            t += [int(x) for x in row[1:row[0] + 2]]
        rounds += 1
        accepted += int(out[:, 0].sum())
    return texts, rounds, accepted


def models(ctx, chats, k, window, sinks, positions, rows_at_once, cache, vocab=512, arithmetic="f32"):
    """A large model, and one that is its first layer with the same embedding and output: a draft that agrees now and then."""
    common = dict(dim=256, n_heads=8, n_kv_heads=2, head_dim=32, ffn=512, vocab=vocab, positions=positions, chats=chats, window=window, sinks=sinks,
                  rows_at_once=max(k + 1, rows_at_once), cache=CACHES[cache], f16=arithmetic == "f16")
    large, small = Stack(ctx, 1, layers=3, **common), Stack(ctx, 1, layers=1, **common)
    small.output = large.output
    return large, small


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--chats", type=int, default=4)
    p.add_argument("--tokens", type=int, default=48)
    p.add_argument("--draft", type=int, default=4)
    p.add_argument("--window", type=int, default=96)
    p.add_argument("--cache", choices=sorted(CACHES), default="q4")
    p.add_argument("--arithmetic", choices=["f32", "f16"], default="f32")
    p.add_argument("--temperature", type=float, default=0.8)
    a = p.parse_args()
    ctx, rows_at_once, sinks = Context(0), 32, 4
    rng = np.random.default_rng(0)
    texts = [rng.integers(0, 512, 20 + 37 * c).tolist() for c in range(a.chats)]
    positions = max(map(len, texts)) + a.tokens * (a.draft + 1) + a.draft + 1  # (a chat runs on until the slowest has its tokens)
    large, small = models(ctx, a.chats, a.draft, a.window, sinks, positions, rows_at_once, a.cache, arithmetic=a.arithmetic)
    began = time.time()
    texts_out, rounds, accepted = generate(ctx, large, small, texts, a.tokens, a.draft, a.temperature, 1, rows_at_once)
    new = sum(len(t) for t in texts_out) - sum(len(t) for t in texts)
    print(f"{a.chats} chats, {new} tokens in {rounds} rounds ({accepted} of {rounds * a.chats * a.draft} drafted tokens accepted), {time.time() - began:.2f} s")
    for t, before in zip(texts_out, texts):
        print(f"  text of {len(before)} tokens continues {t[len(before):][:12]} ...")


if __name__ == "__main__":
    main()
