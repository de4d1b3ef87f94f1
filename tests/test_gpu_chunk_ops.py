"""GPU parity of rope_and_cache, chunk_attention and verify_draft_tokens against plain 64-bit forms.

Tolerances follow from the arithmetic.  With h half a step of the output type (finfo.eps / 2):
  chunk_attention  the result is rounded once (h |o|); the probabilities enter the product with V in 16 bits (h each)
                   and their exponential is good to 2^-12 of itself; a score is a float32 sum of head_dim products
                   (head_dim 2^-24 of the sum of their magnitudes, which moves a probability by as much; twice, for
                   numerator and denominator); with an int8 cache the query times the scales is rounded to fp16
                   (2^-11 of the same sum).  All of it relative to A = sum p |v| / sum p.  With an int8 cache the product
                   runs over the raw values r and (sum p r / sum p + offset) * descale follows: with p' = p (1 + d),
                   |d| <= e, it is off by descale |sum p d r| / sum p <= e * sum p |r| descale / sum p, so A is taken over
                   |r| descale there (the offset carries no error of p).
  rope_and_cache   one rounding (h |y|) of a float32 value that a handful of float32 operations give (8 * 2^-24 of the
                   magnitudes |a c| + |b s|).
"""
import math

import numpy as np
import pytest
import torch

import ms_custom_ops_b200 as ops

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------ chunk_attention
class Chunk:
    """A ragged batch over a paged cache whose unused rows hold NaN (int8: extreme values) and whose unused
    block-table entries point nowhere."""

    def __init__(self, q_lens, ctx, heads=8, kv_heads=2, dim=128, block=16, dtype="bf16", int8=False, layout=0, window=0,
                 offsets=False, seed=0, spare_rows=0, scale=None, blocks=None, freed=True):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q_lens, self.ctx = list(q_lens), list(ctx)
        self.heads, self.kv_heads, self.dim, self.block, self.layout = heads, kv_heads, dim, block, layout
        self.window, self.dtype, self.int8 = window, DT[dtype], int8
        self.scale = 1 / math.sqrt(dim) if scale is None else scale
        need = [-(-c // block) for c in ctx]
        width = max(need + [1]) + 2
        total = sum(need)
        nb = blocks or total + 3
        pool = torch.randperm(nb, generator=g, device="cuda")[:total].cpu()
        if blocks:  # a sparse pool: the last block is among those used
            pool[0] = nb - 1
            pool[1:] = torch.arange(total - 1)
        bad = [-1, nb, 2 ** 31 - 1, -(2 ** 31)]
        tables = torch.tensor([bad[i % 4] for i in range(len(ctx) * width)], dtype=torch.int64).view(len(ctx), width)
        at = 0
        for b, n in enumerate(need):
            tables[b, :n] = pool[at:at + n]
            at += n
        shape = (nb, kv_heads, block, dim) if layout else (nb, block, kv_heads, dim)
        tokens = sum(q_lens)
        self.query = torch.randn(tokens + spare_rows, heads, dim, generator=g, device="cuda").to(self.dtype)
        if int8:
            self.kc = torch.full(shape, -128, dtype=torch.int8, device="cuda")
            self.vc = torch.full(shape, 127, dtype=torch.int8, device="cuda")
        else:
            self.kc = torch.full(shape, float("nan"), dtype=self.dtype, device="cuda")
            self.vc = torch.full(shape, float("nan"), dtype=self.dtype, device="cuda")
        for b, c in enumerate(ctx):
            for cache in (self.kc, self.vc):
                if int8:
                    rows = torch.randint(-128, 128, (c, kv_heads, dim), generator=g, device="cuda", dtype=torch.int8)
                else:
                    rows = torch.randn(c, kv_heads, dim, generator=g, device="cuda").to(self.dtype)
                j = torch.arange(c, device="cuda")
                blk = tables[b].cuda()[j // block]
                if layout:
                    cache[blk, :, j % block] = rows
                else:
                    cache[blk, j % block] = rows
        if window and freed:  # pages that no new token sees any more have been given back
            for b, (ql, c) in enumerate(zip(q_lens, ctx)):
                gone = max(0, c - ql - window + 1) // block if ql else need[b]
                tables[b, :gone] = -1
        self.full_tables = tables
        self.tables = tables.to(torch.int32).cuda()
        ch = kv_heads * dim
        self.scales = {}
        if int8:
            self.scales = dict(k_descale=0.01 + 0.01 * torch.rand(ch, generator=g, device="cuda"),
                               v_descale=0.01 + 0.01 * torch.rand(ch, generator=g, device="cuda"))
            if offsets:
                self.scales["k_offset"] = torch.randint(-20, 20, (ch,), generator=g, device="cuda", dtype=torch.int32)
                self.scales["v_offset"] = torch.randint(-20, 20, (ch,), generator=g, device="cuda", dtype=torch.int32)

    def run(self, **kw):
        return ops.chunk_attention(self.query, self.kc, self.vc, self.tables, torch.tensor(self.q_lens, dtype=torch.int32),
                                   torch.tensor(self.ctx, dtype=torch.int32), qk_scale=self.scale,
                                   window_size=self.window, input_layout=self.layout, **self.scales, **kw)

    def rows_of(self, cache, name, b, lo, c, raw=False):
        """Rows [lo, c) of sequence b in 64 bits, [rows, kv_heads, dim]; `raw`: int8 values without their offset."""
        j = torch.arange(lo, c, device="cuda")
        blk = self.full_tables[b].cuda()[j // self.block]
        x = (cache[blk, :, j % self.block] if self.layout else cache[blk, j % self.block]).double()
        if self.int8:
            shape = (self.kv_heads, self.dim)
            if name + "_offset" in self.scales and not raw:
                x = x + self.scales[name + "_offset"].double().view(shape)
            x = x * self.scales[name + "_descale"].double().view(shape)
        return x

    def expected(self):
        """(output, lse, tolerance of the output, tolerance of lse) in 64 bits."""
        tokens, grp = sum(self.q_lens), self.heads // self.kv_heads
        out = torch.zeros(tokens, self.heads, self.dim, dtype=torch.float64, device="cuda")
        tol, lse = torch.zeros_like(out), torch.full((tokens, self.heads), -math.inf, dtype=torch.float64, device="cuda")
        lse_tol = torch.full_like(lse, 1e-6)
        h = half_step(self.dtype)
        at = 0
        for b, (ql, c) in enumerate(zip(self.q_lens, self.ctx)):
            lo = max(0, c - ql - self.window + 1) if self.window else 0
            lo = min(lo, c)
            if ql and c:
                k, v = self.rows_of(self.kc, "k", b, lo, c), self.rows_of(self.vc, "v", b, lo, c)
                v_mag = self.rows_of(self.vc, "v", b, lo, c, raw=True).abs()
                j = torch.arange(lo, c, device="cuda")
                for t0 in range(0, ql, 1024):
                    t1 = min(ql, t0 + 1024)
                    pos = torch.arange(c - ql + t0, c - ql + t1, device="cuda")
                    seen = j[None] <= pos[:, None]
                    if self.window:
                        seen &= j[None] > pos[:, None] - self.window
                    some = seen.any(1)
                    for hd in range(self.heads):
                        q = self.query[at + t0:at + t1, hd].double()
                        kk, vv = k[:, hd // grp], v[:, hd // grp]
                        s = (q @ kk.T * self.scale).masked_fill(~seen, -math.inf)
                        top = s.amax(1, keepdim=True)
                        p = torch.exp(s - torch.where(some[:, None], top, 0.0))
                        l = p.sum(1, keepdim=True)
                        den = torch.where(some[:, None], l, 1.0)
                        o, a = p @ vv / den, p @ v_mag[:, hd // grp] / den
                        mag = (q.abs() @ kk.abs().T * abs(self.scale)).masked_fill(~seen, 0).amax(1, keepdim=True)
                        ds = mag * (self.dim * 2.0 ** -24 + (2.0 ** -11 if self.int8 else 0.0))
                        out[at + t0:at + t1, hd] = o
                        tol[at + t0:at + t1, hd] = h * o.abs() + (h + 2.0 ** -12 + 2 * ds) * a * 1.01 + 1e-30
                        lse[at + t0:at + t1, hd] = torch.where(some, (top + torch.log(den))[:, 0], -math.inf)
                        lse_tol[at + t0:at + t1, hd] += 2.0 ** -12 + ds[:, 0]
            at += ql
        return out, lse, tol, lse_tol

    def check(self, got=None, lse=None):
        if got is None:
            got, lse = self.run(return_lse=True)
        ops.chunk_attention_check_status()
        tokens = sum(self.q_lens)
        out, want_lse, tol, lse_tol = self.expected()
        got = got[:tokens].double()
        assert torch.isfinite(got).all(), "non-finite output"
        over = ((got - out).abs() - tol).max().item() if tokens else 0.0
        assert over <= 0, f"outside the tolerance by {over:.3e} (largest tolerance {tol.max().item():.3e})"
        if lse is not None:
            lse = lse[:tokens].double()
            assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
            fine = torch.isfinite(want_lse)
            assert ((lse - want_lse).abs() <= lse_tol)[fine].all()


RAGGED = ([5, 1, 0, 33, 1, 130, 17, 64], [5, 300, 40, 33, 1, 517, 129, 1000])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("block,layout", [(16, 0), (128, 0), (32, 1), (64, 1)])
def test_ragged_batch(dtype, dim, block, layout):
    Chunk(*RAGGED, dim=dim, block=block, dtype=dtype, layout=layout, seed=dim + block).check()


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (6, 2), (5, 1), (7, 1), (16, 1), (24, 2), (40, 8), (64, 1),
                                            (100, 1), (128, 1), (200, 1)])
def test_groups(heads, kv_heads):
    Chunk([70, 1, 9], [70, 200, 333], heads=heads, kv_heads=kv_heads, block=32, seed=heads).check()


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 127, 128, 129, 256, 5000])
@pytest.mark.parametrize("dim,layout", [(64, 0), (128, 1)])
def test_window_and_pages_given_back(window, dim, layout):
    Chunk([40, 1, 300, 0, 3], [640, 513, 900, 77, 3], dim=dim, block=16, layout=layout, window=window, seed=window).check()


@pytest.mark.parametrize("q_len", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("past", [0, 1, 63, 64, 127, 128, 129, 255, 1000])
def test_borders(q_len, past):
    Chunk([q_len], [q_len + past], heads=4, kv_heads=1, block=64, seed=q_len * 1000 + past).check()


def test_more_new_tokens_than_cached():
    # the first new tokens stand in front of the cache: nothing to see, zeros
    c = Chunk([10, 300, 4], [3, 140, 0], block=16, dim=64, seed=3)
    out, lse = c.run(return_lse=True)
    c.check(out, lse)
    assert (out[:7] == 0).all() and torch.isinf(lse[:7]).all()
    assert (out[310:] == 0).all()


@pytest.mark.parametrize("dim,block", [(33, 16), (80, 48), (96, 5), (256, 16), (8, 16), (128, 48), (64, 256), (1, 3)])
@pytest.mark.parametrize("layout", [0, 1])
def test_general_shapes(dim, block, layout):
    Chunk([20, 1, 0, 100], [50, 300, 3, 260], heads=6, kv_heads=2, dim=dim, block=block, layout=layout, seed=dim).check()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("dim,block", [(128, 16), (128, 128), (64, 32), (40, 16)])
def test_int8_cache(dtype, offsets, dim, block):
    Chunk([70, 1, 0, 33, 200], [70, 700, 9, 257, 600], dim=dim, block=block, dtype=dtype, int8=True, offsets=offsets,
          seed=dim + block).check()


def test_int8_scales_of_very_different_size():
    # a channel's scale may be thousands of times another's: the query times the scales stays in range
    c = Chunk([70, 1], [200, 700], block=32, int8=True, dtype="bf16", seed=11)
    f = torch.logspace(-4, 2, c.scales["k_descale"].numel(), device="cuda")
    c.scales["k_descale"] = c.scales["k_descale"] * f[torch.randperm(f.numel(), device="cuda")]
    c.scale = 0.002
    c.check()


@pytest.mark.parametrize("q_lens,ctx", [([1], [70001]), ([3, 1, 1], [20000, 33, 40001]), ([200], [20011]), ([16], [9000])])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_contexts(q_lens, ctx, dim):
    Chunk(q_lens, ctx, heads=8, kv_heads=2, dim=dim, block=128, seed=sum(ctx)).check()


@pytest.mark.parametrize("window", [700, 5000])
def test_windows_over_long_contexts(window):
    Chunk([1, 3, 200, 1], [20000, 9000, 15000, 130], heads=8, kv_heads=2, block=64, window=window, seed=window).check()
    Chunk([129, 1], [9000, 12001], heads=2, kv_heads=2, dim=64, block=16, window=window, seed=window).check()


@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (8, 8), (40, 1), (64, 2)])
@pytest.mark.parametrize("offsets", [False, True])
def test_few_rows_over_long_int8_contexts(heads, kv_heads, offsets):
    Chunk([4, 1, 2, 1], [9000, 20000, 131, 128], heads=heads, kv_heads=kv_heads, block=128, int8=True, offsets=offsets,
          seed=heads).check()


@pytest.mark.parametrize("which", ["query", "out"])
def test_rows_that_are_not_aligned(which):
    # copies of 16 bytes cannot start on them: the general kernel takes the call
    c = Chunk([20, 1], [300, 1000], block=16, seed=33)
    base = torch.empty(c.query.numel() + 1, dtype=c.query.dtype, device="cuda")
    view = base[1:].view(c.query.shape)
    if which == "query":
        view.copy_(c.query)
        c.query = view
        c.check()
    else:
        out, lse = c.run(out=view, return_lse=True)
        assert out is view
        c.check(out, lse)


def test_large_scores_and_negative_scale():
    c = Chunk([100], [400], dtype="fp16", scale=3.0, seed=5)
    c.check()
    Chunk([100], [400], dtype="bf16", scale=-0.2, seed=6).check()
    Chunk([100], [400], dtype="bf16", scale=0.0, seed=7).check()


def test_growing_scores():
    # keys that grow along the context: the running maximum moves at every tile
    c = Chunk([64], [1500], heads=4, kv_heads=1, block=128, seed=8, dtype="bf16")
    c.query[:] = c.query.abs()
    ramp = torch.linspace(0.01, 3, 1500, device="cuda")
    j = torch.arange(1500, device="cuda")
    blk = c.full_tables[0].cuda()[j // 128]
    c.kc[blk, j % 128] = (c.kc[blk, j % 128].abs().float() * ramp[:, None, None]).to(torch.bfloat16)
    c.check()


@pytest.mark.parametrize("batch", [65, 1000])
def test_many_sequences(batch):
    rng = np.random.default_rng(batch)
    q = rng.integers(0, 4, batch)
    Chunk(q.tolist(), (q + rng.integers(0, 60, batch)).tolist(), heads=4, kv_heads=2, dim=64, block=16, seed=batch).check()


def test_a_sequence_does_not_depend_on_the_others():
    c = Chunk([70, 1, 300, 5], [400, 9000, 1300, 2000], block=32, seed=21)
    out, lse = c.run(return_lse=True)
    at = 0
    for b, q in enumerate(c.q_lens):
        one, one_lse = ops.chunk_attention(c.query[at:at + q].clone(), c.kc, c.vc, c.tables[b:b + 1].clone(), [q], [c.ctx[b]],
                                           qk_scale=c.scale, return_lse=True)
        assert torch.equal(one.view(torch.int16), out[at:at + q].view(torch.int16))
        assert torch.equal(one_lse, lse[at:at + q])
        at += q


def test_rows_behind_the_last_sequence():
    c = Chunk([3, 70], [50, 90], spare_rows=9, seed=31)
    out, lse = c.run(return_lse=True)
    assert (out[73:] == 0).all() and torch.isinf(lse[73:]).all()
    c.check(out, lse)
    mine = torch.full_like(c.query, 7.0)
    assert c.run(out=mine) is mine
    assert (mine[73:] == 7.0).all()
    assert torch.equal(mine[:73], out[:73])
    with pytest.raises(ValueError):
        c.run(out=c.query)


def test_no_new_tokens():
    c = Chunk([0, 0], [10, 0], spare_rows=2, seed=1)
    assert (c.run() == 0).all()
    e = ops.chunk_attention(c.query[:0], c.kc, c.vc, c.tables[:0], [], [])
    assert e.shape == (0, 8, 128)


def test_block_ids_outside_the_cache_are_counted():
    c = Chunk([40, 1], [130, 300], seed=41)
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.run(oob_count=count)
    assert count.item() == 0
    c.tables[0, 1] = -5
    c.tables[1, 3] = c.kc.shape[0]
    c.kc.nan_to_num_(), c.vc.nan_to_num_()
    out = c.run(oob_count=count)
    assert count.item() >= 2 and torch.isfinite(out).all()


def test_agrees_with_paged_attention_on_single_tokens():
    c = Chunk([1] * 6, [1, 17, 300, 4000, 129, 9000], heads=16, kv_heads=4, block=128, dtype="fp16", seed=51)
    out, lse = c.run(return_lse=True)
    other, other_lse = ops.paged_attention_with_lse(c.query, c.kc, c.vc, c.tables.clamp(0, c.kc.shape[0] - 1), c.ctx,
                                                    q_head_num=16, kv_head_num=4, qk_scale=c.scale)
    _, _, tol, lse_tol = c.expected()
    assert ((out.double() - other.double()).abs() <= 2 * tol).all()
    assert ((lse - other_lse).abs() <= 2 * lse_tol).all()


def test_halves_of_a_context_merge_by_fa_update():
    # the older cache without the chunk (a window-free call per half would mask by position, so the old half
    # is a call of single tokens), merged with the chunk's own part
    c = Chunk([1], [1000], heads=8, kv_heads=2, block=16, seed=61)
    whole, lse = c.run(return_lse=True)
    a, la = ops.chunk_attention(c.query, c.kc, c.vc, c.tables, [1], [608], qk_scale=c.scale, return_lse=True)
    b, lb = ops.chunk_attention(c.query, c.kc, c.vc, c.tables[:, 38:].contiguous(), [1], [392], qk_scale=c.scale,
                                return_lse=True)
    m = ops.fa_update(torch.stack([la.view(-1), lb.view(-1)]), torch.stack([a.float().view(-1, 128), b.float().view(-1, 128)]),
                      0, 2).view(1, 8, 128)
    _, _, tol, _ = c.expected()
    assert ((m.double() - whole.double()).abs() <= 3 * tol).all()


def test_other_streams_at_once():
    cs = [Chunk([200, 1], [3000, 20000], block=64, seed=70 + i) for i in range(3)]
    want = [c.run().clone() for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[], [], []]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cs, streams)):
            with torch.cuda.stream(s):
                got[i].append(c.run())
    torch.cuda.synchronize()
    for i in range(3):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_captured_graphs_replayed_at_once():
    cs = [Chunk([100, 1], [2000, 30000], block=64, seed=80 + i) for i in range(2)]
    want = [c.run().clone() for c in cs]
    graphs, outs = [], []
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run())
        graphs.append(g)
    for c in cs:  # other inputs before the replay, the captured ones again for the last
        c.query.neg_()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert not torch.equal(outs[0], want[0])
    for c in cs:
        c.query.neg_()
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_offsets_past_32_bits():
    # 2^31 elements are 4 GB of a bf16 cache: the last block lies behind them
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    blocks = (2 ** 31) // (128 * 8 * 128) + 5
    Chunk([20], [300], heads=16, kv_heads=8, block=128, blocks=blocks, seed=91).check()


# ------------------------------------------------------------------------------------------ rope_and_cache
def rope_case(tokens=37, heads=8, kv_heads=2, dim=128, rotary=None, block=16, dtype="bf16", int8=False, layout=0,
              interleaved=False, norm=False, fused=False, offsets=False, seed=0, positions=500, extra=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rotary = dim if rotary is None else rotary
    dt = DT[dtype]
    rows = torch.randn(tokens, heads + 2 * kv_heads + extra, dim, generator=g, device="cuda").to(dt)
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:heads + 2 * kv_heads]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    nb = tokens // block + 3
    shape = (nb, kv_heads, block, dim) if layout else (nb, block, kv_heads, dim)
    cd = torch.int8 if int8 else dt
    c = dict(q=q, k=k, v=v, dim=dim, rotary=rotary, block=block, layout=layout, interleaved=interleaved, dt=dt,
             kc=torch.randn(shape, generator=g, device="cuda").to(cd), vc=torch.randn(shape, generator=g, device="cuda").to(cd),
             slots=torch.randperm(nb * block, generator=g, device="cuda")[:tokens].to(torch.int32),
             positions=torch.randint(0, positions, (tokens,), generator=g, device="cuda", dtype=torch.int32),
             cos_sin=torch.randn(positions, rotary, generator=g, device="cuda"), eps=1e-5, qw=None, kw=None, scales={})
    if norm:
        c["qw"] = torch.randn(dim, generator=g, device="cuda").to(dt)
        c["kw"] = torch.randn(dim, generator=g, device="cuda").to(dt)
    ch = kv_heads * dim
    if int8:
        c["scales"] = dict(k_descale=0.02 + 0.03 * torch.rand(ch, generator=g, device="cuda"),
                           v_descale=0.02 + 0.03 * torch.rand(ch, generator=g, device="cuda"))
        if offsets:
            c["scales"]["k_offset"] = torch.randint(-9, 9, (ch,), generator=g, device="cuda", dtype=torch.int32)
            c["scales"]["v_offset"] = torch.randint(-9, 9, (ch,), generator=g, device="cuda", dtype=torch.int32)
    return c


def rope_run(c, **kw):
    return ops.rope_and_cache(c["q"], c["k"], c["v"], c["kc"], c["vc"], c["slots"], c["positions"], c["cos_sin"],
                              q_weight=c["qw"], k_weight=c["kw"], eps=c["eps"], interleaved=c["interleaved"],
                              input_layout=c["layout"], **c["scales"], **kw)


def rope_expected(c):
    """(rotated queries, key cache, value cache, tolerances of the three) in 64 bits (int8 caches: steps)."""
    r, half = c["rotary"], c["rotary"] // 2
    at = c["positions"].long().clamp(0, c["cos_sin"].shape[0] - 1)
    cos, sin = c["cos_sin"].double()[at, None, :half], c["cos_sin"].double()[at, None, half:]
    h = half_step(c["dt"])

    def turn(x, w):
        x = x.double()
        if w is not None:
            x = x * w.double() / torch.sqrt(x.square().mean(-1, keepdim=True) + c["eps"])
        y, mag = x.clone(), x.abs()
        i = torch.arange(half, device="cuda")
        a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        mag[..., a] = (x[..., a] * cos).abs() + (x[..., b] * sin).abs()
        mag[..., b] = (x[..., b] * cos).abs() + (x[..., a] * sin).abs()
        return y, mag * 8 * 2.0 ** -24

    ok = (c["positions"] >= 0) & (c["positions"] < c["cos_sin"].shape[0])
    q, qt = turn(c["q"], c["qw"])
    q = torch.where(ok[:, None, None], q, 0.0)
    k, kt = turn(c["k"], c["kw"])
    v, vt = c["v"].double(), torch.zeros_like(c["v"], dtype=torch.float64)
    nslots = c["kc"].shape[0] * c["block"]
    keep = (c["slots"] >= 0) & (c["slots"] < nslots) & ok
    slot = c["slots"][keep].long()
    caches, tols = [], []
    for cache, x, t, name in ((c["kc"], k, kt, "k"), (c["vc"], v, vt, "v")):
        want = cache.double().clone()
        tol = torch.zeros_like(want)
        if c["scales"]:
            shape = x.shape[1:]
            d = c["scales"][name + "_descale"].double().view(shape)
            y = x / d
            near = ((y - y.floor() - 0.5).abs() <= t / d + y.abs() * 2.0 ** -23).double()  # next to a tie: either neighbour
            x = torch.clamp(torch.round(y) - c["scales"].get(name + "_offset", torch.zeros(1, device="cuda")).double()
                            .view(shape if name + "_offset" in c["scales"] else (1,)), -128, 127)
            t = near
        else:
            t = t + h * x.abs() + torch.finfo(c["dt"]).smallest_normal * torch.finfo(c["dt"]).eps
        if c["layout"]:
            want[slot // c["block"], :, slot % c["block"]] = x[keep]
            tol[slot // c["block"], :, slot % c["block"]] = t[keep]
        else:
            want[slot // c["block"], slot % c["block"]] = x[keep]
            tol[slot // c["block"], slot % c["block"]] = t[keep]
        caches.append(want)
        tols.append(tol)
    qt = qt + h * q.abs() + torch.finfo(c["dt"]).smallest_normal * torch.finfo(c["dt"]).eps
    return q, *caches, qt, *tols


def rope_check(c, **kw):
    q, kc, vc, qt, kt, vt = rope_expected(c)
    got = rope_run(c, **kw)
    assert got.is_contiguous()
    for name, g, w, t in (("query", got, q, qt), ("key cache", c["kc"], kc, kt), ("value cache", c["vc"], vc, vt)):
        over = ((g.double() - w).abs() - t * 1.001).max().item() if g.numel() else 0
        assert over <= 0, f"{name}: outside the tolerance by {over:.3e}"
    return got


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (64, 64), (64, 32), (256, 256), (256, 64), (128, 32),
                                        (128, 96), (128, 2), (128, 0), (96, 96), (80, 40), (33, 10), (512, 512), (40, 40),
                                        (128, 126), (192, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_shapes(dtype, dim, rotary, interleaved, norm):
    rope_check(rope_case(dim=dim, rotary=rotary, dtype=dtype, interleaved=interleaved, norm=norm, layout=norm, seed=dim + rotary))


@pytest.mark.parametrize("tokens", [1, 2, 3, 64, 511, 3000])
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (1, 1), (7, 1), (5, 5), (0, 3), (64, 4)])
def test_rope_sizes(tokens, heads, kv_heads):
    rope_check(rope_case(tokens=tokens, heads=heads, kv_heads=kv_heads, fused=True, norm=tokens % 2 == 0, seed=tokens))


@pytest.mark.parametrize("fused,extra", [(True, 0), (True, 3), (False, 0)])
@pytest.mark.parametrize("dim", [128, 36])
def test_rope_strides(fused, extra, dim):
    rope_check(rope_case(tokens=50, dim=dim, rotary=dim // 2 // 2 * 2, fused=fused, extra=extra, seed=extra))


def test_rope_rows_that_are_not_aligned():
    c = rope_case(tokens=20, fused=False, norm=True)
    for n in ("q", "k", "v"):
        base = torch.empty(c[n].numel() + 1, dtype=c[n].dtype, device="cuda")
        base[1:] = c[n].flatten()
        c[n] = base[1:].view(c[n].shape)
    rope_check(c)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("dim,rotary,interleaved,norm", [(128, 128, False, False), (128, 64, True, True), (64, 64, False, True),
                                                         (40, 20, True, False)])
def test_rope_int8(dtype, offsets, dim, rotary, interleaved, norm):
    rope_check(rope_case(tokens=70, dim=dim, rotary=rotary, dtype=dtype, int8=True, offsets=offsets, interleaved=interleaved,
                         norm=norm, fused=True, seed=dim))


def test_rope_padding_and_indices_out_of_range():
    c = rope_case(tokens=60, norm=True, seed=5)
    nslots = c["kc"].shape[0] * c["block"]
    c["slots"][::5] = -1
    c["slots"][7], c["slots"][8] = nslots, 2 ** 31 - 1
    c["slots"][11] = -(2 ** 31)
    c["positions"][21], c["positions"][22], c["positions"][23] = -1, 500, 2 ** 31 - 1
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = rope_check(c, oob_count=count)
    assert count.item() == 5
    assert (out[21:24] == 0).all()


def test_rope_without_tokens():
    c = rope_case(tokens=4)
    for n in ("q", "k", "v", "slots", "positions"):
        c[n] = c[n][:0]
    before = c["kc"].clone()
    assert rope_run(c).shape == (0, 8, 128) and torch.equal(before, c["kc"])


def test_rope_equals_reshape_and_cache_without_rotation():
    c = rope_case(tokens=90, rotary=0, seed=9)
    kc, vc = c["kc"].clone(), c["vc"].clone()
    ops.reshape_and_cache(c["k"].reshape(90, -1), c["v"].reshape(90, -1), kc, vc, c["slots"])
    assert torch.equal(rope_run(c), c["q"])
    assert torch.equal(kc, c["kc"]) and torch.equal(vc, c["vc"])


def test_rope_slots_past_32_bits():
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    c = rope_case(tokens=6, heads=8, kv_heads=8, block=128)
    nb = (2 ** 31) // (128 * 8 * 128) + 3
    c["kc"] = torch.zeros(nb, 128, 8, 128, dtype=torch.bfloat16, device="cuda")
    c["vc"] = torch.zeros_like(c["kc"])
    c["slots"] = (nb * 128 - 1 - torch.arange(6, device="cuda") * 3).to(torch.int32)
    small = dict(c, kc=torch.zeros(2, 128, 8, 128, dtype=torch.bfloat16, device="cuda"))
    small["vc"] = torch.zeros_like(small["kc"])
    small["slots"] = c["slots"] - (nb - 2) * 128
    rope_check(small)
    rope_run(c)
    assert torch.equal(c["kc"][-2:], small["kc"]) and torch.equal(c["vc"][-2:], small["vc"])
    assert not c["kc"][0].any()


# ------------------------------------------------------------------------------------------ verify_draft_tokens
def verify_case(batch, drafts, vocab, dtype="fp32", given=True, noise=0.7, seed=0, peak=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[dtype]
    logits = peak * torch.randn(batch, drafts + 1, vocab, generator=g, device="cuda")
    target = torch.softmax(logits, -1).to(dt)
    draft = torch.softmax(logits[:, :drafts] + noise * torch.randn(batch, drafts, vocab, generator=g, device="cuda"), -1).to(dt)
    if drafts:
        tokens = torch.multinomial(draft.reshape(-1, vocab).float(), 1, generator=g).view(batch, drafts).to(torch.int32)
    else:
        tokens = torch.empty(batch, 0, dtype=torch.int32, device="cuda")
    return target, draft if given else None, tokens, torch.rand(batch, drafts + 1, generator=g, device="cuda")


def verify_expected(target, draft, tokens, uniform, lens=None):
    batch, drafts = tokens.shape
    vocab = target.shape[2]
    t, u = target.double().cpu().numpy(), uniform.double().cpu().numpy()
    d = None if draft is None else draft.double().cpu().numpy()
    tok = tokens.cpu().numpy()
    lens = [drafts] * batch if lens is None else lens.clamp(0, drafts).tolist()
    out, count = np.full((batch, drafts + 1), -1, np.int32), np.zeros(batch, np.int32)
    for b in range(batch):
        n = 0
        while n < lens[b]:
            x = tok[b, n]
            if not 0 <= x < vocab or not u[b, n] * (d[b, n, x] if d is not None else 1.0) < t[b, n, x]:
                break
            n += 1
        p = np.maximum(t[b, n], 0)
        w = p
        if n < lens[b]:
            q = np.zeros(vocab)
            if d is not None:
                q = d[b, n]
            elif 0 <= tok[b, n] < vocab:
                q[tok[b, n]] = np.inf
            w = np.maximum(p - q, 0)
            if not w.sum() > 0:
                w = p
        c = np.cumsum(w)
        out[b, :n] = tok[b, :n]
        if c[-1] > 0:
            out[b, n] = int(np.argmax(c > u[b, drafts] * c[-1]))
        count[b] = n
    return out, count


def verify_check(args, lens=None):
    tokens, accepted = ops.verify_draft_tokens(*args, draft_lens=lens)
    want, count = verify_expected(*args, lens=lens)
    assert np.array_equal(accepted.cpu().numpy(), count)
    assert np.array_equal(tokens.cpu().numpy(), want)
    return tokens, accepted


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 1000, 4096, 32000, 50257, 128256])
@pytest.mark.parametrize("given", [True, False])
def test_verify_vocabularies(dtype, vocab, given):
    verify_check(verify_case(9, 3, vocab, dtype, given, seed=vocab))


@pytest.mark.parametrize("batch,drafts", [(1, 0), (1, 1), (3, 0), (2, 40), (130, 2), (5, 33), (1, 64)])
def test_verify_sizes(batch, drafts):
    verify_check(verify_case(batch, drafts, 3001, noise=0.05, seed=batch + drafts))


def test_verify_draft_lens():
    args = verify_case(8, 5, 5000, noise=0.0, seed=4)
    lens = torch.tensor([0, 1, 2, 3, 4, 5, 9, -3], dtype=torch.int32, device="cuda")
    _, accepted = verify_check(args, lens)
    assert accepted.tolist() == [0, 1, 2, 3, 4, 5, 5, 0]  # equal distributions: every draft is taken


def test_verify_bad_token_ids():
    target, draft, tokens, uniform = verify_case(6, 3, 400, noise=0.0, seed=5)
    tokens[0, 0], tokens[1, 1], tokens[2, 2] = -1, 400, 2 ** 31 - 1
    tokens[3, 1] = -(2 ** 31)
    verify_check((target, draft, tokens, uniform))
    verify_check((target, None, tokens, uniform * 0.001))


def test_verify_draws():
    # weights of few, exactly known places: both ends, the border at a sum that is met exactly, nothing at all
    target = torch.zeros(6, 1, 10000, device="cuda")
    target[0, 0, 9999] = 1.0
    target[1, 0, 0] = 1.0
    target[2, 0, [5, 5000, 9000]] = torch.tensor([0.25, 0.25, 0.5], device="cuda")
    target[3] = target[2]
    target[4] = target[2]
    uniform = torch.tensor([[0.999], [0.0], [0.25], [0.4999], [0.9999]], device="cuda")
    uniform = torch.cat([uniform, torch.tensor([[0.5]], device="cuda")])
    none = torch.empty(6, 0, dtype=torch.int32, device="cuda")
    tokens, accepted = ops.verify_draft_tokens(target, None, none, uniform)
    assert tokens[:, 0].tolist() == [9999, 0, 5000, 5000, 9000, -1]
    assert accepted.tolist() == [0] * 6


def test_verify_rest_that_is_nowhere_positive():
    # the draft covers the target: the difference is nowhere positive, the draw is the target's own
    target = torch.full((2, 2, 3000), 1 / 4096.0, device="cuda")
    draft = torch.full((2, 1, 3000), 1.0, device="cuda")
    tok = torch.tensor([[5], [7]], dtype=torch.int32, device="cuda")
    uniform = torch.tensor([[0.9, 0.5], [0.00001, 0.1]], device="cuda")
    tokens, accepted = verify_check((target, draft, tok, uniform))
    assert accepted.tolist() == [0, 1] and tokens[0, 0].item() == 1500


def test_verify_in_a_graph_and_on_a_stream():
    args = verify_case(16, 4, 20000, seed=7)
    want, count = ops.verify_draft_tokens(*args)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got, n = ops.verify_draft_tokens(*args)
    got.zero_()
    g.replay()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other, _ = ops.verify_draft_tokens(*args)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(n, count) and torch.equal(other, want)


# ------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("layout", [0, 1])
def test_a_step_of_chunks(int8, layout):
    """Two steps of three sequences: rows of a fused projection are rotated and cached, the chunk attends to everything
    cached so far; against attention over the rotated rows in 64 bits."""
    if int8 and layout:
        pytest.skip("one layout is enough for the int8 cache")
    g = torch.Generator(device="cuda").manual_seed(17)
    heads, kv, dim, block, dt = 8, 2, 128, 16, torch.bfloat16
    nb = 60
    shape = (nb, kv, block, dim) if layout else (nb, block, kv, dim)
    kc = torch.zeros(shape, dtype=torch.int8 if int8 else dt, device="cuda")
    vc = torch.zeros_like(kc)
    tables = torch.randperm(nb, generator=g, device="cuda")[:45].view(3, 15).to(torch.int32)
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    ang = torch.arange(300, device="cuda", dtype=torch.float64)[:, None] * inv
    cos_sin = torch.cat([ang.cos(), ang.sin()], 1).float()
    scales = {}
    if int8:
        scales = dict(k_descale=torch.full((kv * dim,), 0.03, device="cuda"), v_descale=torch.full((kv * dim,), 0.03, device="cuda"))
    ctx = [0, 0, 0]
    weight = (1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).to(dt)
    for q_lens in ([70, 33, 129], [5, 1, 64]):
        rows = torch.randn(sum(q_lens), heads + 2 * kv, dim, generator=g, device="cuda").to(dt)
        pos = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, q_lens)]).to(torch.int32).cuda()
        seq = torch.cat([torch.full((n,), b) for b, n in enumerate(q_lens)]).cuda()
        slots = tables[seq, pos.long() // block] * block + pos % block
        q = ops.rope_and_cache(rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:], kc, vc, slots, pos, cos_sin,
                               q_weight=weight, k_weight=weight, input_layout=layout, **scales)
        ctx = [c + n for c, n in zip(ctx, q_lens)]
        out, lse = ops.chunk_attention(q, kc, vc, tables, q_lens, ctx, qk_scale=dim ** -0.5, input_layout=layout,
                                       return_lse=True, **scales)
        c = Chunk.__new__(Chunk)
        c.q_lens, c.ctx, c.heads, c.kv_heads, c.dim, c.block, c.layout = q_lens, ctx, heads, kv, dim, block, layout
        c.window, c.dtype, c.int8, c.scale, c.scales = 0, dt, int8, dim ** -0.5, scales
        c.query, c.kc, c.vc, c.full_tables = q, kc, vc, tables.long().cpu()
        c.check(out, lse)
        # the cached keys are the rotated ones
        x = rows[:, heads:heads + kv].double()
        x = x * weight.double() / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        t = cos_sin.double()[pos.long()][:, None]
        a, b = x[..., :64], x[..., 64:]
        x = torch.cat([a * t[..., :64] - b * t[..., 64:], b * t[..., :64] + a * t[..., 64:]], -1)
        s = slots.long()
        stored = (kc[s // block, :, s % block] if layout else kc[s // block, s % block]).double()
        if int8:
            assert ((stored * 0.03 - x.clamp(-128 * 0.03, 127 * 0.03)).abs() <= 0.015 * 1.001).all()
        else:
            assert ((stored - x).abs() <= x.abs() * 2.0 ** -8 + 1e-5).all()


def test_a_speculative_step():
    """Drafted tokens of three sequences through the cache, the attention and the check, the accepted ones kept."""
    g = torch.Generator(device="cuda").manual_seed(23)
    heads, kv, dim, block, vocab, drafts = 4, 1, 64, 16, 2000, 3
    kc = torch.zeros(20, block, kv, dim, dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    tables = torch.arange(18, device="cuda", dtype=torch.int32).view(3, 6)
    cos_sin = torch.randn(100, dim, generator=g, device="cuda")
    proj = torch.randn(heads * dim, vocab, generator=g, device="cuda") * 0.05
    past = [10, 0, 31]
    for b, n in enumerate(past):
        kc.view(-1, kv, dim)[b * 96:b * 96 + n] = torch.randn(n, kv, dim, generator=g, device="cuda").half()
        vc.view(-1, kv, dim)[b * 96:b * 96 + n] = torch.randn(n, kv, dim, generator=g, device="cuda").half()
    for step in range(3):
        q_lens = [drafts + 1] * 3
        rows = torch.randn(12, heads + 2 * kv, dim, generator=g, device="cuda").half()
        pos = torch.cat([torch.arange(n, n + 4) for n in past]).to(torch.int32).cuda()
        slots = torch.cat([b * 96 + torch.arange(n, n + 4) for b, n in enumerate(past)]).to(torch.int32).cuda()
        q = ops.rope_and_cache(rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:], kc, vc, slots, pos, cos_sin)
        out = ops.chunk_attention(q, kc, vc, tables, q_lens, [n + 4 for n in past], qk_scale=dim ** -0.5)
        target = torch.softmax(out.float().view(3, 4, heads * dim) @ proj, -1)
        draft = torch.softmax(torch.log(target[:, :3]) + 0.1 * torch.randn(3, 3, vocab, generator=g, device="cuda"), -1)
        tokens = torch.multinomial(draft.view(9, vocab), 1, generator=g).view(3, 3).to(torch.int32)
        uniform = torch.rand(3, 4, generator=g, device="cuda")
        _, accepted = verify_check((target.contiguous(), draft.contiguous(), tokens, uniform))
        past = [n + 1 + a for n, a in zip(past, accepted.tolist())]
