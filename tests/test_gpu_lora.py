"""GPU: low-rank adapters against the formula in 64 bits.

Tolerance.  With e half a step of the data's type: h is an fp32 sum rounded once, so it is off by e |h| and by the accumulation,
whose K / 16 steps each keep sixteen products and the sum so far to 2^-22 of their magnitudes at worst; the expand adds R / 16
such steps, and the result is rounded once, e |out|.
"""
import pytest
import torch

from helpers import same_bits

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def _case(T, K, sizes, R, L, dtype, seed, ranks=None):
    g = torch.Generator().manual_seed(seed)
    S, N = len(sizes), sum(sizes)
    x, base = torch.randn(T, K, generator=g).to(dtype), torch.randn(T, N, generator=g).to(dtype)
    A = (torch.randn(L, S * R, K, generator=g) * K ** -0.5).to(dtype)
    B = (torch.randn(L, N, R, generator=g) * 0.2).to(dtype)
    ids = torch.randint(-1, L, (T,), generator=g).int()
    if ranks is None:
        ranks = [[R, max(1, R // 2), max(1, R - 3), 1][a % 4] for a in range(L)]
    ranks = torch.tensor(ranks).int()
    # what lies behind a rank is never used
    for a in range(L):
        r = int(ranks[a])
        A.view(L, S, R, K)[a, :, max(r, 0):] = float("nan")
        B[a, :, max(r, 0):] = float("nan")
    return x, base, A, B, ids, ranks, torch.rand(L, generator=g) * 3 - 1


def _exact(x, base, A, B, ids, ranks, scal, sizes):
    """(h, out, tolerance of h, tolerance of out) in 64 bits."""
    T, K = x.shape
    L, N, R = B.shape
    S, f = len(sizes), torch.finfo(x.dtype)
    e, step, tiny = f.eps / 2, 2.0 ** -22, f.smallest_normal * f.eps / 2
    h, h_tol = torch.zeros(T, S * R, dtype=torch.float64), torch.zeros(T, S * R, dtype=torch.float64)
    out = base.double().clone() if base is not None else torch.zeros(T, N, dtype=torch.float64)
    tol = torch.zeros(T, N, dtype=torch.float64)
    for a in range(L):
        rows, r = (ids == a).nonzero().flatten(), int(min(ranks[a], R))
        if r <= 0 or not len(rows):
            continue
        at = 0
        for s, n in enumerate(sizes):
            A64, B64 = A[a, s * R:s * R + r].double(), B[a, at:at + n, :r].double()
            hh = x[rows].double() @ A64.T
            ht = e * hh.abs() + (K / 16 + 4) * step * (x[rows].double().abs() @ A64.abs().T) + tiny
            h[rows, s * R:s * R + r], h_tol[rows, s * R:s * R + r] = hh, ht
            out[rows, at:at + n] += float(scal[a]) * hh @ B64.T
            tol[rows, at:at + n] += abs(float(scal[a])) * (ht + (R / 16 + 4) * step * hh.abs()) @ B64.abs().T * (1 + e)
            at += n
    return h, out, h_tol, tol * (1 + e) + e * out.abs() + 2.0 ** -23 * out.abs() + tiny


def _close(got, want, tol):
    bad = ~((got.cpu().double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist(), got.cpu()[bad][:3], want[bad][:3], tol[bad][:3])


CASES = [
    (1, 8, [8], 8, 1), (1, 8192, [8192], 16, 4), (2, 64, [64], 16, 3), (7, 72, [72, 8], 8, 2), (8, 1000, [200, 8, 8], 40, 5),
    (9, 256, [128, 0, 64], 24, 3), (16, 4096, [64, 64], 64, 2), (17, 520, [264], 128, 4), (33, 96, [40, 24, 16, 8], 256, 3),
    (129, 1024, [256, 64, 64], 64, 33), (300, 264, [136], 32, 1000), (515, 512, [320, 64, 64], 64, 3), (1000, 2048, [512, 512], 16, 2),
    (2049, 320, [192], 8, 40), (700, 136, [72, 72], 128, 2), (640, 200, [48, 16], 256, 2), (513, 8, [32, 8], 72, 2),
    (16, 256, [512, 64], 16, 2), (5, 264, [2048, 1024, 1024], 8, 2), (33, 520, [64], 32, 2), (3, 8200, [16384], 24, 9), (12, 1032, [8, 72], 16, 3),
    (255, 192, [40], 16, 2), (256, 192, [40], 16, 2), (263, 128, [16, 24], 24, 11), (264, 128, [16, 24], 24, 11), (257, 648, [264, 8], 64, 10),
]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T,K,sizes,R,L", CASES)
def test_apply(T, K, sizes, R, L, dtype):
    from sglang_b200.layers.lora import LoRABatch, apply_lora, lora_expand, lora_shrink
    c = _case(T, K, sizes, R, L, dtype, T + K + R)
    x, base, A, B, ids, ranks, scal = c
    h_want, want, h_tol, tol = _exact(*c, sizes)
    xd, bd, Ad, Bd = x.cuda(), base.cuda(), A.cuda(), B.cuda()
    batch = LoRABatch(ids.cuda(), ranks.cuda(), scal.cuda())
    h = lora_shrink(xd, Ad, batch, len(sizes))
    _close(h, h_want, h_tol)
    out = torch.full_like(bd, float("nan"))
    assert apply_lora(bd, xd, Ad, Bd, batch, output_sizes=sizes, out=out) is not None
    _close(out, want, tol)
    assert same_bits(bd, base)
    assert same_bits(lora_expand(h, Bd, batch, bd, sizes, out=torch.empty_like(bd)), out)
    # in place; tokens without an adapter untouched, whatever they hold
    none = (ids < 0).cuda()
    bd[none] = float("nan")
    got = apply_lora(bd, xd, Ad, Bd, batch, output_sizes=tuple(sizes))
    assert got.data_ptr() == bd.data_ptr() and same_bits(got[~none], out[~none]) and got[none].isnan().all()
    # no base: zeros
    _, want0, _, tol0 = _exact(x, None, A, B, ids, ranks, scal, sizes)
    _close(apply_lora(None, xd, Ad, Bd, batch, output_sizes=sizes), want0, tol0)


@pytest.mark.parametrize("seed", range(4))
def test_runs_of_neighbouring_tokens(seed):
    """Requests of several tokens: tiles whose tokens are neighbours, have gaps in different places, or end early."""
    from sglang_b200.layers.lora import LoRABatch, apply_lora
    g = torch.Generator().manual_seed(seed)
    lens = [[130, 64, 96, 40, 17, 8, 200, 145], [1, 127, 129, 16, 48, 32, 260], [500, 3, 5, 9, 33, 65, 256], [24] * 30][seed]
    which = torch.tensor([(3 * i) % 4 - 1 for i in range(len(lens))])[torch.randperm(len(lens), generator=g)]
    T, K, sizes, R, L = sum(lens), 456, [72, 40], 32, 3
    x, base, A, B, _, ranks, scal = _case(T, K, sizes, R, L, BF, seed)
    ids = torch.repeat_interleave(which, torch.tensor(lens)).int()
    batch = LoRABatch(ids.cuda(), ranks.cuda(), scal.cuda())
    _, want, _, tol = _exact(x, base, A, B, ids, ranks, scal, sizes)
    _close(apply_lora(base.cuda(), x.cuda(), A.cuda(), B.cuda(), batch, sizes), want, tol)


@pytest.mark.parametrize("T", [3, 300])
def test_nobody_has_an_adapter(T):
    from sglang_b200.layers.lora import LoRABatch, apply_lora, lora_shrink
    x, base, A, B, _, ranks, scal = _case(T, 128, [64], 16, 2, BF, T)
    batch = LoRABatch(torch.full((T,), -1, dtype=torch.int32, device="cuda"), ranks.cuda(), scal.cuda())
    xd, bd = x.cuda(), base.cuda()
    for _ in range(3):
        assert same_bits(apply_lora(bd, xd, A.cuda(), B.cuda(), batch), base)
        assert same_bits(apply_lora(bd, xd, A.cuda(), B.cuda(), batch, out=torch.full_like(bd, 5.0)), base)
        assert (apply_lora(None, xd, A.cuda(), B.cuda(), batch) == 0).all()
        assert (lora_shrink(xd, A.cuda(), batch) == 0).all()


def test_several_streams_at_once():
    """Calls of one batch on several streams, each with its own tokens and output."""
    from sglang_b200.layers.lora import LoRABatch, apply_lora
    for T, R in ((6, 16), (6, 32), (300, 32)):
        cases = [_case(T, 512, [128, 64], R, 3, BF, 50 + i) for i in range(4)]
        x0, _, A, B, ids, ranks, scal = cases[0]
        Ad, Bd = A.cuda(), B.cuda()
        batch = LoRABatch(ids.cuda(), ranks.cuda(), scal.cuda())
        xs, bases = [c[0].cuda() for c in cases], [c[1].cuda() for c in cases]
        alone = [apply_lora(b.clone(), x, Ad, Bd, batch, [128, 64]) for x, b in zip(xs, bases)]
        torch.cuda.synchronize()
        streams, outs = [torch.cuda.Stream() for _ in cases], [torch.empty_like(b) for b in bases]
        for _ in range(20):
            for s, x, b, o in zip(streams, xs, bases, outs):
                with torch.cuda.stream(s):
                    apply_lora(b, x, Ad, Bd, batch, [128, 64], out=o)
        torch.cuda.synchronize()
        for a, o in zip(alone, outs):
            assert same_bits(a, o)


def test_plans_of_several_threads():
    """Many and few adapters planned by two threads at once: the plan's kernel needs 143 KB of shared memory or 54 KB."""
    import threading

    from sglang_b200.layers.lora import LoRABatch
    failed = []

    def work(L):
        with torch.cuda.stream(torch.cuda.Stream()):
            ids = torch.zeros(8, dtype=torch.int32, device="cuda")
            batch = LoRABatch(ids, torch.ones(L, dtype=torch.int32, device="cuda"), torch.ones(L, device="cuda"))
            try:
                for _ in range(20000):
                    batch.update()
            except RuntimeError as e:
                failed.append((L, str(e)))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(L,)) for L in (1024, 400)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_strided_views_and_odd_ids():
    """x and base as columns of wider tensors; ids outside the buffers and ranks of 0 or below count as no adapter; a rank
    above R counts as R."""
    from sglang_b200.layers.lora import LoRABatch, apply_lora
    T, K, sizes, R, L = 50, 128, [64, 32], 16, 4
    x, base, A, B, ids, ranks, scal = _case(T, K, sizes, R, L, BF, 5, ranks=[16, 0, -3, 99])
    ids[:4] = torch.tensor([4, 1 << 30, -(1 << 31), -2])
    wide_x, wide = torch.randn(T, 3 * K).to(BF).cuda(), torch.full((T, 200), 7.0, dtype=BF, device="cuda")
    wide_x[:, K:2 * K], wide[:, 8:104] = x.cuda(), base.cuda()
    batch = LoRABatch(ids.cuda(), ranks.cuda(), scal.cuda())
    out = apply_lora(wide[:, 8:104], wide_x[:, K:2 * K], A.cuda(), B.cuda(), batch, sizes)
    _, want, _, tol = _exact(x, base, A, B, ids, ranks, scal, sizes)
    _close(out, want, tol)
    idle = (ids < 0) | (ids >= L) | (ids == 1) | (ids == 2)
    assert same_bits(out.cpu()[idle], base[idle])
    assert (wide[:, :8] == 7).all() and (wide[:, 104:] == 7).all()


def test_a_token_s_result_depends_on_its_own_row_only():
    """Infinities and NaN in one token leave every other token's bits alone; so does the company a token is in."""
    from sglang_b200.layers.lora import LoRABatch, apply_lora
    for T, R in ((10, 16), (24, 32), (270, 32), (700, 32)):
        x, base, A, B, ids, ranks, scal = _case(T, 320, [96, 32], R, 3, BF, T)
        one = lambda xx, rows: apply_lora(base[rows].cuda(), xx[rows].cuda(), A.cuda(), B.cuda(),  # noqa: E731
                                          LoRABatch(ids[rows].cuda(), ranks.cuda(), scal.cuda()), [96, 32])
        every = torch.arange(T)
        clean = one(x, every)
        spoilt = x.clone()
        spoilt[3], spoilt[T - 2] = float("nan"), float("inf")
        got = one(spoilt, every)
        keep = torch.ones(T, dtype=torch.bool)
        keep[3] = keep[T - 2] = False
        assert same_bits(got[keep.cuda()], clean[keep.cuda()])
        order = torch.randperm(T, generator=torch.Generator().manual_seed(1))
        assert same_bits(one(x, order), clean[order.cuda()])


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T,R,L,ranks", [(3, 16, 2, [5, 12]), (40, 64, 4, [64, 33, 1, 31]), (300, 32, 3, [4, 17, 32]), (700, 64, 2, [3, 63]),
                                         (600, 128, 2, [97, 127]), (513, 256, 2, [250, 129])])
def test_expand_uses_nothing_behind_a_rank(T, R, L, ranks, dtype):
    """h from elsewhere, with infinities and NaN behind every adapter's rank and in the rows of tokens without one."""
    from sglang_b200.layers.lora import LoRABatch, lora_expand
    sizes = [72, 24]
    x, base, A, B, ids, ranks, scal = _case(T, 64, sizes, R, L, dtype, T + R, ranks=ranks)
    h = torch.randn(T, 2, R, generator=torch.Generator().manual_seed(R)).to(dtype)
    out = base.double().clone()
    tol = torch.zeros_like(out)
    step, e = 2.0 ** -22, torch.finfo(dtype).eps / 2
    for a in range(L):
        rows, r = (ids == a).nonzero().flatten(), int(ranks[a])
        h[rows, :, r:] = float("nan") if a % 2 else float("inf")
        for s, (at, n) in enumerate(((0, 72), (72, 24))):
            hh, bb = h[rows, s, :r].double(), B[a, at:at + n, :r].double()
            out[rows, at:at + n] += float(scal[a]) * hh @ bb.T
            # fp32 sums of products of 16-bit numbers, as at the top of this file; the result is rounded once
            tol[rows, at:at + n] = abs(float(scal[a])) * (R / 16 + 4) * step * hh.abs() @ bb.abs().T * (1 + e)
    h[ids < 0] = float("nan")
    got = lora_expand(h.view(T, 2 * R).cuda(), B.cuda(), LoRABatch(ids.cuda(), ranks.cuda(), scal.cuda()), base.cuda(), sizes)
    _close(got, out, tol + e * out.abs() + 2.0 ** -23 * out.abs() + torch.finfo(dtype).smallest_normal * e)


@pytest.mark.parametrize("T,R", [(3, 16), (40, 64), (300, 64)])
def test_h_beyond_the_range_of_fp16(T, R):
    """x A^T is rounded to x's type before it is scaled: beyond 65504 it is infinite in fp16, for its own token only; bf16 holds it."""
    from sglang_b200.layers.lora import LoRABatch, apply_lora, lora_shrink
    for dtype in (F16, BF):
        x, base, A, B, ids, ranks, scal = _case(T, 512, [64], R, 1, dtype, T, ranks=[R])
        ids[:] = 0
        A[0, 3], x[1] = 2.0, 100.0                             # h[1, 3] = 102400
        B.fill_(0.25)
        scal.fill_(2.0 ** -10)
        batch = LoRABatch(ids.cuda(), ranks.cuda(), scal.cuda())
        h = lora_shrink(x.cuda(), A.cuda(), batch).cpu()
        out = apply_lora(base.cuda(), x.cuda(), A.cuda(), B.cuda(), batch).cpu()
        rest = torch.arange(T) != 1
        assert h[rest].isfinite().all() and out[rest].isfinite().all()
        assert h[1, 3] == (float("inf") if dtype == F16 else 102400.0)
        assert out[1].isfinite().all() if dtype == BF else not out[1].isfinite().any()


def test_segments_and_update():
    from sglang_b200.layers.lora import LoRABatch, apply_lora
    T, sizes = 90, [64]
    x, base, A, B, _, ranks, scal = _case(T, 64, sizes, 16, 3, F16, 9)
    which, lens = torch.tensor([2, -1, 0, 2, 1]), torch.tensor([30, 10, 0, 49, 1])
    batch = LoRABatch.from_segments(which.cuda(), lens.cuda(), T, ranks.cuda(), scal.cuda())
    ids = torch.repeat_interleave(which, lens).int()
    out = apply_lora(base.cuda(), x.cuda(), A.cuda(), B.cuda(), batch)
    _, want, _, tol = _exact(x, base, A, B, ids, ranks, scal, sizes)
    _close(out, want, tol)
    # the ids of the next batch, written in place
    ids = ids.flip(0).contiguous()
    batch.token_adapters.copy_(ids)
    batch.update()
    out = apply_lora(base.cuda(), x.cuda(), A.cuda(), B.cuda(), batch)
    _, want, _, tol = _exact(x, base, A, B, ids, ranks, scal, sizes)
    _close(out, want, tol)


@pytest.mark.parametrize("T,live", [(90, 57), (90, 0), (90, 200), (600, 411)])
def test_a_padded_batch_of_segments(T, live):
    """Requests that hold fewer tokens than the batch, or more: also planned and run in a graph, for the lengths at its replay."""
    from sglang_b200.layers.lora import LoRABatch, apply_lora
    x, base, A, B, _, ranks, scal = _case(T, 64, [64], 16, 3, F16, 9)
    which, lens = torch.tensor([2, 1, -1, 0]), torch.tensor([live // 2, live // 5, live // 5, live - live // 2 - 2 * (live // 5)])
    ids = torch.full((T + live,), -1, dtype=torch.int32)
    ids[:live] = torch.repeat_interleave(which, lens).int()
    ids = ids[:T]
    _, want, _, tol = _exact(x, base, A, B, ids, ranks, scal, [64])
    xd, bd, Ad, Bd, rd, sd, wd, ld = (t.cuda() for t in (x, base, A, B, ranks, scal, which, lens))
    out = apply_lora(bd, xd, Ad, Bd, LoRABatch.from_segments(wd, ld, T, rd, sd), out=torch.empty_like(bd))
    _close(out, want, tol)
    assert same_bits(out[ids < 0], base[ids < 0])
    later, got = torch.zeros_like(ld), torch.empty_like(bd)
    LoRABatch.from_segments(wd, later, T, rd, sd)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        apply_lora(bd, xd, Ad, Bd, LoRABatch.from_segments(wd, later, T, rd, sd), out=got)
    later.copy_(ld)
    g.replay()
    assert same_bits(got, out)


@pytest.mark.parametrize("T,R", [(5, 16), (5, 32), (260, 32), (600, 32)])
def test_captured_and_replayed_on_a_side_stream(T, R):
    """Planning, shrink and expand in one graph; new tokens and ids are copied in before each replay.  Two graphs share nothing
    but the weights."""
    from sglang_b200.layers.lora import LoRABatch, apply_lora
    K, sizes, L = 256, [64, 64], 6
    _, _, A, B, _, ranks, scal = _case(1, K, sizes, R, L, BF, 1)
    Ad, Bd, graphs = A.cuda(), B.cuda(), []
    for _ in range(2):
        st = dict(x=torch.zeros(T, K, dtype=BF, device="cuda"), base=torch.zeros(T, 128, dtype=BF, device="cuda"),
                  ids=torch.zeros(T, dtype=torch.int32, device="cuda"), out=torch.empty(T, 128, dtype=BF, device="cuda"))
        batch = LoRABatch(st["ids"], ranks.cuda(), scal.cuda())
        apply_lora(st["base"], st["x"], Ad, Bd, batch, sizes, out=st["out"])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            batch.update()
            apply_lora(st["base"], st["x"], Ad, Bd, batch, sizes, out=st["out"])
        graphs.append((g, st, batch))
    cases = []
    for i, (g, st, _) in enumerate(graphs * 2):
        x, base, _, _, ids, _, _ = _case(T, K, sizes, R, L, BF, 100 + i)
        for name, value in (("x", x), ("base", base), ("ids", ids)):
            st[name].copy_(value)
        g.replay()
        cases.append((x, base, ids, st["out"].clone()))
    for x, base, ids, out in cases:
        _, want, _, tol = _exact(x, base, A, B, ids, ranks, scal, sizes)
        _close(out, want, tol)


def test_empty_batches():
    from sglang_b200.layers.lora import LoRABatch, apply_lora, lora_shrink
    z = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731
    batch = LoRABatch(torch.zeros(0, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda"), torch.ones(2, device="cuda"))
    assert apply_lora(z(0, 16), z(0, 64), z(2, 8, 64), z(2, 16, 8), batch).shape == (0, 16)
    assert lora_shrink(z(0, 64), z(2, 8, 64), batch).shape == (0, 8)
    batch = LoRABatch(torch.zeros(3, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda"), torch.ones(2, device="cuda"))
    assert (lora_shrink(z(3, 0), z(2, 8, 0), batch) == 0).all()
    assert (apply_lora(None, z(3, 64), z(2, 8, 64), z(2, 16, 8), batch) == 0).all()


def test_buffers_beyond_32_bits():
    """A of 4.3 GB: the last adapter lies behind offset 2^32."""
    from sglang_b200.layers.lora import LoRABatch, lora_shrink
    L, R, K = 33, 256, 262144
    A = torch.empty(L, R, K, dtype=BF, device="cuda")
    A[L - 1].normal_(std=K ** -0.5, generator=torch.Generator(device="cuda").manual_seed(0))
    x = torch.randn(3, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(BF)
    batch = LoRABatch(torch.full((3,), L - 1, dtype=torch.int32, device="cuda"), torch.full((L,), R, dtype=torch.int32, device="cuda"),
                      torch.ones(L, device="cuda"))
    want = x.double() @ A[L - 1].double().T
    size = x.double().abs() @ A[L - 1].double().abs().T
    assert ((lora_shrink(x, A, batch).double() - want).abs() <= 2 ** -8 * want.abs() + (K / 16 + 4) * 2.0 ** -22 * size).all()
