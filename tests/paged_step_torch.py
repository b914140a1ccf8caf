"""A whole paged step on torch's streams and in a torch graph (run by test_gpu_paged_step.py, as
python -m tests.paged_step_torch captured | streams)."""
import sys

import numpy as np
import torch

from rapidllm_amd import hip
from rapidllm_amd.hip import call

V, NQ, NKV, HD, ROT, THETA = 97, 4, 2, 64, 32, 1e4
F32, F16 = 0, 1


class Device:
    """One step's buffers for direct calls on a stream."""

    def __init__(self, seed, B=3, R=5):
        self.t = torch
        r = np.random.default_rng(seed)
        self.B, self.R, n = B, R, B * R
        self.page, self.width = 16, 8
        dev = lambda a, t: torch.tensor(np.asarray(a), dtype=t, device="cuda")  # noqa: E731
        self.k = torch.zeros(2, B * self.width, NKV, self.page, HD, dtype=torch.float16, device="cuda")
        self.v = torch.zeros_like(self.k)
        self.cache = hip.RlPagedCache(self.k.data_ptr(), self.v.data_ptr(), self.k[0].numel(), 2, B * self.width,
                                      self.page, NKV, HD, F16)
        self.table = dev(r.permutation(B * self.width).reshape(B, self.width), torch.int32)
        self.start = dev(np.arange(B + 1) * R, torch.int32)
        self.y = torch.zeros(n, NQ + 2 * NKV, HD, device="cuda")
        self.pos, self.slots = dev(np.zeros(n), torch.int32), dev(np.zeros(n), torch.int64)
        self.mask, self.par = dev(np.zeros((n, 1)), torch.int64), dev(np.zeros(n), torch.int32)
        self.toks, self.u = dev(np.zeros(n), torch.int32), torch.zeros(n, device="cuda")
        self.ctx = dev(np.zeros(B), torch.int32)
        self.W = dev(r.standard_normal((NQ * HD, V)), torch.float32)
        f32 = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.q, self.out, self.prob = f32(n, NQ, HD), f32(n, NQ, HD), f32(n)
        self.logits = f32(n, V)
        self.pick, self.path, self.n, self.nxt, self.ctx2 = i32(n), i32(B, R), i32(B), i32(B), i32(B)
        L = hip.lib()
        self.ws = torch.zeros(L.rl_hip_tree_attn_workspace_bytes(NQ, NKV, HD, B, R), dtype=torch.uint8, device="cuda")
        self.ws2 = torch.zeros(L.rl_hip_sample_workspace_bytes(n, V), dtype=torch.uint8, device="cuda")

    def fill(self, seed):
        """New inputs, in place: contexts, trees, rows, numbers, and what the cache holds."""
        r, t = np.random.default_rng(seed), self.t
        ctx = r.integers(0, 100, self.B)
        parents, bits, depth = [], [], []
        for b in range(self.B):
            own = []
            for i in range(self.R):
                p = int(r.integers(0, i)) if i else -1
                parents.append(p)
                own.append((own[p][0] | 1 << i, own[p][1] + 1) if i else (1, 0))
            bits += [o[0] for o in own]
            depth += [o[1] for o in own]
        seq, row = np.repeat(np.arange(self.B), self.R), np.tile(np.arange(self.R), self.B)
        where = ctx[seq] + row
        table = self.table.cpu().numpy()
        put = lambda d, a: d.copy_(t.tensor(np.asarray(a), dtype=d.dtype).reshape(d.shape))  # noqa: E731
        put(self.ctx, ctx)
        put(self.par, parents)
        put(self.mask, bits)
        put(self.pos, ctx[seq] + np.array(depth))
        put(self.slots, table[seq, where // self.page].astype(np.int64) * self.page + where % self.page)
        put(self.toks, r.integers(0, 3, self.B * self.R))
        put(self.u, r.random(self.B * self.R))
        put(self.y, r.standard_normal(tuple(self.y.shape)))
        put(self.k, r.standard_normal(tuple(self.k.shape)))
        put(self.v, r.standard_normal(tuple(self.v.shape)))
        t.cuda.synchronize()

    def step(self):
        s = self.t.cuda.current_stream().cuda_stream
        n, ld, y = self.B * self.R, (NQ + 2 * NKV) * HD, self.y.data_ptr()
        call("rl_hip_paged_append", self.cache, 1, F32, y, ld, HD, y + 4 * NQ * HD, ld, HD, y + 4 * (NQ + NKV) * HD, ld,
             HD, None, None, 1, 1e-6, ROT, THETA, self.pos.data_ptr(), self.slots.data_ptr(), n, NQ, self.q.data_ptr(), s)
        call("rl_hip_tree_attn", self.cache, 1, F32, self.q.data_ptr(), NQ * HD, HD, None, 0, 0, self.table.data_ptr(),
             self.width, self.ctx.data_ptr(), self.start.data_ptr(), self.B, n, self.R, self.mask.data_ptr(), 1, NQ,
             HD ** -0.5, self.out.data_ptr(), self.ws.data_ptr(), self.ws.numel(), s)
        self.t.mm(self.out.view(n, -1), self.W, out=self.logits)
        call("rl_hip_sample_rows", F32, self.logits.data_ptr(), V, n, V, None, None, None, None, self.u.data_ptr(),
             self.pick.data_ptr(), self.prob.data_ptr(), self.ws2.data_ptr(), self.ws2.numel(), s)
        # tokens of a small vocabulary, so that paths are taken
        self.pick.remainder_(3)
        call("rl_hip_tree_accept", self.cache, self.table.data_ptr(), self.width, self.ctx.data_ptr(),
             self.start.data_ptr(), self.B, n, self.par.data_ptr(), self.toks.data_ptr(), self.pick.data_ptr(),
             self.path.data_ptr(), self.R, self.n.data_ptr(), self.nxt.data_ptr(), self.ctx2.data_ptr(), s)

    def outputs(self):
        return [x.clone() for x in (self.q, self.out, self.prob, self.pick, self.path, self.n, self.nxt, self.ctx2,
                                    self.k, self.v)]


def captured():
    """The whole step in a graph: every replay, over new contexts, trees and cache contents, gives what
    the eager calls give; eager work and synchronisation in between."""
    d = Device(1)
    d.fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        d.step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        d.step()
    taken = 0
    for seed in range(1, 6):
        d.fill(seed)
        d.step()
        torch.cuda.synchronize()
        want = d.outputs()
        d.fill(seed)
        for x in (d.q, d.out, d.prob, d.pick, d.path, d.n, d.nxt, d.ctx2):
            x.zero_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(d.outputs(), want):
            assert torch.equal(a, b)
        taken += int(d.n.sum())
    assert taken > 5 * d.B  # more than the roots


def streams():
    """Two steps on two streams, each with its own cache and workspaces, many times over."""
    ds = [Device(s) for s in (1, 2)]
    want = []
    for i, d in enumerate(ds):
        d.fill(10 + i)
        d.step()
        torch.cuda.synchronize()
        want.append(d.outputs())
        d.fill(10 + i)
    streams = [torch.cuda.Stream() for _ in ds]
    for _ in range(20):
        for d, s in zip(ds, streams):
            with torch.cuda.stream(s):
                # the caches move on, so only the first outputs of each pass are compared
                d.step()
    torch.cuda.synchronize()
    for i, d in enumerate(ds):
        d.fill(10 + i)
    for d, s in zip(ds, streams):
        with torch.cuda.stream(s):
            d.step()
    torch.cuda.synchronize()
    for d, w in zip(ds, want):
        for a, b in zip(d.outputs(), w):
            assert torch.equal(a, b)


if __name__ == "__main__":
    {"captured": captured, "streams": streams}[sys.argv[1]]()
    print("STEP_OK")
