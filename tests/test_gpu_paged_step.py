"""The paged operators together, as a serving step uses them: append, attention of the drafted
trees, sampling, acceptance; eagerly, captured into a graph, and on several streams."""
import os
import subprocess
import sys

import numpy as np
import pytest

from rapidllm_amd import ops
from rapidllm_amd.ops import BF16, F16, F32
from tests.test_gpu_paged import Step, agree, norm_rope, rounded

pytestmark = pytest.mark.gpu

V, NQ, NKV, HD, ROT, THETA = 97, 4, 2, 64, 32, 1e4


class Toy:
    """One attention layer over token embeddings: logits = attention(q, k, v of the tokens) @ W."""

    def __init__(self, seed):
        r = np.random.default_rng(seed)
        self.q, self.k, self.v = (r.standard_normal((V, h, HD)).astype(np.float32) for h in (NQ, NKV, NKV))
        self.qn, self.kn = (r.standard_normal(HD).astype(np.float32) * 0.2 for _ in range(2))
        self.W = (r.standard_normal((NQ * HD, V)) * 0.7).astype(np.float32)

    def sequential(self, prompt, n, temperature, u):
        """Tokens one by one in 64 bits; u[p] picks the token at position p."""
        toks = list(prompt)
        while len(toks) < len(prompt) + n:
            p = np.arange(len(toks))
            K = rounded(norm_rope(self.k[toks], self.kn, p, ROT, THETA)[0], F16).astype(np.float64)
            v = rounded(self.v[toks], F16).astype(np.float64)
            q = norm_rope(self.q[toks[-1:]], self.qn, p[-1:], ROT, THETA)[0][0]
            o = []
            for h in range(NQ):
                s = K[:, h // (NQ // NKV)] @ q[h] / np.sqrt(HD)
                w = np.exp(s - s.max())
                o.append(w @ v[:, h // (NQ // NKV)] / w.sum())
            z = np.concatenate(o) @ self.W.astype(np.float64)
            if temperature == 0:
                toks.append(int(z.argmax()))
            else:
                w = np.exp((z - z.max()) / temperature)
                c = np.cumsum(w)
                toks.append(int(np.searchsorted(c, float(u[len(toks)]) * c[-1], side="right")))
        return toks


@pytest.mark.parametrize("page,temperature", [(1, 0.0), (16, 0.0), (16, 1.0), (64, 0.7)])
def test_tree_steps_generate_what_single_steps_do(gpu, page, temperature):
    """Three sequences, trees with the right continuation among wrong ones (or without it): every step
    keeps the path that single steps would have taken."""
    toy, r = Toy(1), np.random.default_rng(page)
    B, new = 3, 25
    u = r.random((B, 200)).astype(np.float32)
    prompts = [list(r.integers(0, V, n)) for n in (1, 17, 40)]
    want = [toy.sequential(p, new, temperature, u[b]) for b, p in enumerate(prompts)]
    width = -(-(40 + new + 40) // page)
    cache = ops.PagedCache(B * width, page, NKV, HD)
    cache.fill(np.full(cache.shape, np.nan), np.full(cache.shape, np.nan))
    table = r.permutation(B * width).reshape(B, width).astype(np.int32)

    def append(toks, b, pos, where):
        slots = table[b, where // page].astype(np.int64) * page + where % page
        return ops.paged_append(cache, 0, toy.q[toks], toy.k[toks], toy.v[toks], pos, slots, toy.qn, toy.kn,
                                rotary_dim=ROT, theta=THETA)

    got, ctx = [list(p) for p in prompts], np.array([len(p) - 1 for p in prompts])
    for b, p in enumerate(prompts):
        if len(p) > 1:
            append(np.array(p[:-1]), b, np.arange(len(p) - 1), np.arange(len(p) - 1))
    steps = 0
    while any(len(g) < len(w) for g, w in zip(got, want)):
        steps += 1
        toks, parents, depth, seq, mask, start = [], [], [], [], [], [0]
        for b in range(B):
            if len(got[b]) >= len(want[b]):  # done: takes no part
                start.append(len(toks))
                continue
            base, t, par, dep = len(toks), [got[b][-1]], [-1], [0]
            ahead = want[b][len(got[b]):]
            good = 0  # node of the right continuation so far
            for i in range(1, int(r.integers(2, 12))):
                d = dep[good]
                if good == len(t) - 1 and d < len(ahead) and r.random() < 0.7 or r.random() < 0.3 and d < len(ahead):
                    t.append(ahead[d]); par.append(good); dep.append(d + 1); good = i
                else:
                    p = int(r.integers(0, i))
                    t.append(int(r.integers(0, V))); par.append(p); dep.append(dep[p] + 1)
            bits = []
            for i, p in enumerate(par):
                bits.append((bits[p] if i else 0) | 1 << i)
            toks += t; parents += par; depth += dep; seq += [b] * len(t); mask += bits
            start.append(base + len(t))
        seq, depth = np.array(seq), np.array(depth)
        row = np.concatenate([np.arange(b - a) for a, b in zip(start, start[1:])])
        pos, where = ctx[seq] + depth, ctx[seq] + row
        q = append(np.array(toks), seq, pos, where)
        out = ops.tree_attn(cache, 0, q, table, ctx, start, np.array(mask, np.uint64)[:, None])
        z = out.reshape(len(toks), -1).astype(np.float64) @ toy.W
        pick, _ = ops.sample_rows(z, u[seq, pos + 1], temperature=temperature)
        path, n, nxt, ctx2 = ops.tree_accept(cache, table, ctx, start, parents, toks, pick, 16)
        for b in range(B):
            a = [toks[start[b] + i] for i in path[b] if i >= 0]
            got[b] += (a[1:] + [int(nxt[b])]) if n[b] else []
            assert ctx2[b] == ctx[b] + n[b]
        ctx = ctx2.astype(int)
    for g, w in zip(got, want):
        assert g[:len(w)] == w
    assert steps < new  # some drafts were taken


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B", [65, 130, 200])
def test_many_sequences(gpu, dtype, B):
    """More sequences than a wave has lanes, some without rows, some without context."""
    r = np.random.default_rng(B)
    ctx = [int(c) for c in r.choice([0, 5, 31, 64, 130], B)]
    rows = [int(n) for n in r.choice([0, 1, 2], B, p=[0.3, 0.4, 0.3])]
    s = Step(B, dtype, 4, 2, 64, 16, ctx, rows)
    agree(s.run(), *s.want(None, False))
    mask = s.tree_mask()
    agree(s.run(mask, True), *s.want(mask, True))


def test_one_long_sequence_among_short_ones(gpu):
    """Work is dealt by length: the long one's positions go to many workgroups."""
    s = Step(5, F32, 6, 1, 128, 64, [9, 6000, 0, 40], [2, 3, 1, 2])
    agree(s.run(), *s.want(None, False))


@pytest.mark.parametrize("what", ["captured", "streams"])
def test_step_under_torch(gpu, what):
    """Graph capture and streams come from torch, whose HIP runtime is a process's only one when it is
    loaded first: a process of its own."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-m", "tests.paged_step_torch", what], cwd=root, capture_output=True, text=True,
                       timeout=110)
    assert p.returncode == 0 and "STEP_OK" in p.stdout, p.stdout[-2000:] + p.stderr[-3000:]
