"""GPU: head norms with the rotation, and the e4m3 key/value cache written and read, against the formulas in 64 bits.

Tolerances.  A result y is computed in fp32 and rounded once: half a step of its type, |y| eps / 2, and the fp32 arithmetic: the
sum of D squares in some order (relative error below D / 2 steps of 2^-24 after the square root), the root, the two products
and the rotation (16 steps are more than all of those), relative to |a cos| + |b sin|.
"""
import pytest
import torch

from helpers import same_bits
from oracle import block_fp8_oracle as O

pytestmark = pytest.mark.gpu
BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _table(rows, rot, base=10000.0):
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _exact(x, w, pos, table, neox, eps):
    """(y, the magnitude that its fp32 error is relative to), in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    y, size = x.clone(), x.abs()
    if table is not None:
        half = table.shape[1] // 2
        c, s = table.double()[pos, None, :half], table.double()[pos, None, half:]
        a = torch.arange(half) if neox else 2 * torch.arange(half)
        b = a + (half if neox else 1)
        xa, xb = x[..., a], x[..., b]
        y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
        size[..., a], size[..., b] = (xa * c).abs() + (xb * s).abs(), (xb * c).abs() + (xa * s).abs()
    return y, size


def _steps(D):
    return (D / 2 + 16) * 2.0 ** -24


def _close(got, y, size, D):
    f = torch.finfo(got.dtype)
    tol = (1 + 2 * _steps(D)) * f.eps / 2 * y.abs() + 2 * _steps(D) * size + f.smallest_normal * f.eps / 2
    bad = (got.cpu().double() - y).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist())


def _inputs(T, Hq, Hkv, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g) * torch.exp2(torch.randn(Hq + 2 * Hkv, 1, generator=g))
    qkv = qkv.to(dtype)
    if T > 1:
        qkv[T // 2, 0] = 0                                    # a head of zeros
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype) for _ in range(2)]
    return qkv, w


def _split(qkv, Hq, Hkv):
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]


def _cache(pages, page, H, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = [(torch.randn(pages, page, H, D, generator=g) * 100).clamp(-448, 448).to(F8).cuda() for _ in range(2)]
    return codes + [torch.rand(pages, page, H, generator=g).cuda() for _ in range(2)]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,neox", [
    (1, 64, 8, 128, 128, True), (1, 1, 1, 16, 16, False), (2, 5, 1, 48, 32, True), (3, 7, 2, 80, 80, True),
    (17, 8, 8, 64, 32, False), (65, 12, 3, 96, 96, True), (33, 4, 4, 192, 64, True), (129, 3, 1, 256, 256, False),
    (700, 64, 8, 128, 128, True), (1500, 32, 4, 128, 64, False), (9, 0, 2, 32, 16, True), (12, 3, 2, 64, 48, False),
    (21, 5, 1, 96, 80, False), (14, 2, 2, 112, 64, True), (6, 9, 2, 240, 16, True),
])
def test_norm_rope(T, Hq, Hkv, D, rot, neox, dtype):
    from sglang_b200.layers.rotary_embedding import qk_norm_rope
    qkv, (qw, kw) = _inputs(T, Hq, Hkv, D, dtype, T + D)
    pos = torch.randint(0, 5000, (T,), generator=torch.Generator().manual_seed(T))
    pos[0], table = 4999, _table(5000, rot)
    dev = qkv.cuda()
    q, k, _ = _split(dev, Hq, Hkv)
    for weights in ((qw, kw), (None, kw), (None, None)):
        on = [w.cuda() if w is not None else None for w in weights]
        qo, ko = qk_norm_rope(q, k, pos.cuda(), table.cuda(), *on, norm_eps=1e-5, is_neox=neox)
        assert qo.is_contiguous() and qo.shape == q.shape and ko.shape == k.shape
        _close(qo, *_exact(qkv[:, :Hq], weights[0], pos, table, neox, 1e-5), D)
        _close(ko, *_exact(qkv[:, Hq:Hq + Hkv], weights[1], pos, table, neox, 1e-5), D)
    assert same_bits(dev, qkv)
    # norm alone, int32 positions, in place: the same bits
    qn, kn = qk_norm_rope(q, k, None, None, qw.cuda(), kw.cuda())
    _close(qn, *_exact(qkv[:, :Hq], qw, pos, None, neox, 1e-6), D)
    _close(kn, *_exact(qkv[:, Hq:Hq + Hkv], kw, pos, None, neox, 1e-6), D)
    out = qk_norm_rope(q, k, pos.int().cuda(), table.cuda(), is_neox=neox, q_out=q, k_out=k)
    assert out[0].data_ptr() == q.data_ptr() and same_bits(q, qo) and same_bits(k, ko)
    assert same_bits(dev[:, Hq + Hkv:], qkv[:, Hq + Hkv:])


def test_norm_rope_padding_and_positions_outside_the_table():
    from sglang_b200.layers.rotary_embedding import qk_norm_rope
    qkv, (qw, kw) = _inputs(6, 4, 2, 64, BF, 3)
    pos = torch.tensor([0, -1, 7, 8, -(1 << 40), 1 << 40])
    table = _table(8, 64).cuda()
    q, k, _ = _split(qkv.cuda(), 4, 2)
    qo, ko = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
    qk_norm_rope(q, k, pos.cuda(), table, qw.cuda(), kw.cuda(), q_out=qo, k_out=ko)
    for out, x, w in ((qo, qkv[:, :4], qw), (ko, qkv[:, 4:6], kw)):
        y, size = _exact(x[[0, 2]], w, pos[[0, 2]], table.cpu(), True, 1e-6)
        _close(out[[0, 2]], y, size, 64)
        assert (out[[1, 4]] == 9.0).all() and out[[3, 5]].isnan().all()


@pytest.mark.parametrize("dtype", [BF, F16])
def test_a_table_without_rows_lacks_every_position(dtype):
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8, qk_norm_rope_store_kv_fp8
    from sglang_b200.layers.rotary_embedding import qk_norm_rope
    qkv, (qw, kw) = _inputs(3, 4, 2, 64, dtype, 3)
    q, k, v = _split(qkv.cuda(), 4, 2)
    pos, table = torch.tensor([0, -1, 7]).cuda(), torch.empty(0, 64, device="cuda")
    for w in ((qw.cuda(), kw.cuda()), (None, None)):
        for neox in (True, False):
            qo, ko = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
            qk_norm_rope(q, k, pos, table, *w, is_neox=neox, q_out=qo, k_out=ko)
            for out in (qo, ko):
                assert out[[0, 2]].isnan().all() and (out[1] == 9.0).all()
    cache = _cache(1, 4, 2, 64)
    out = qk_norm_rope_store_kv_fp8(q, k, v, pos, table, *cache, torch.arange(3).cuda())
    kl, vl = load_kv_fp8(*cache, torch.tensor([[0]]).int().cuda(), torch.tensor([0, 3]).int().cuda(), 3)
    assert out[[0, 2]].isnan().all() and kl[[0, 2]].isnan().all() and not vl.isnan().any()


@pytest.mark.parametrize("queries,weights", [(2, True), (2, False), (0, True), (0, False)])
def test_padding_without_a_rotation(queries, weights):
    """A negative position marks a token as padding whether or not there is a table."""
    from sglang_b200.layers.quantization.kv_cache import qk_norm_rope_store_kv_fp8
    from sglang_b200.layers.rotary_embedding import qk_norm_rope
    T, H, D = 5, 3, 64
    pos = torch.tensor([7, -1, 0, -5, 1 << 20], device="cuda")
    idle = (pos < 0).cpu()
    q, k, v = (torch.randn(T, h, D, device="cuda").to(BF) for h in (queries, H, H))
    w = torch.ones(D, device="cuda", dtype=BF) if weights else None
    qo, ko = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
    qk_norm_rope(q, k, pos, None, w, w, q_out=qo, k_out=ko)
    assert (qo[pos < 0] == 9).all() and (ko[pos < 0] == 9).all()
    want_q, want_k = qk_norm_rope(q, k, None, None, w, w)
    assert torch.equal(qo[pos >= 0], want_q[pos >= 0]) and torch.equal(ko[pos >= 0], want_k[pos >= 0])
    caches = []
    for p in (pos, None):
        cache = [torch.zeros(2, 4, H, D, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
        cache += [torch.full((2, 4, H), 3.0, device="cuda") for _ in range(2)]
        qk_norm_rope_store_kv_fp8(q, k, v, p, None, *cache, torch.arange(T, device="cuda"), w, w)
        caches.append([c.cpu() for c in cache])
    for got, want in zip(*caches):
        got, want = (c.view(torch.uint8) if c.dtype != torch.float32 else c for c in (got, want))
        got, want = got.reshape(8, H, -1)[:T], want.reshape(8, H, -1)[:T]
        assert torch.equal(got[~idle], want[~idle])
        assert (got[idle] == (3 if got.dtype == torch.float32 else 0)).all()


def test_infinities_and_nan_stay_in_their_head():
    from sglang_b200.layers.rotary_embedding import qk_norm_rope
    qkv, (qw, kw) = _inputs(4, 4, 2, 128, BF, 5)
    clean = qkv.clone()
    qkv[1, 2, 3], qkv[2, 4, 7] = float("inf"), float("nan")
    pos, table = torch.arange(4).cuda(), _table(16, 128).cuda()
    run = lambda x: qk_norm_rope(x[:, :4], x[:, 4:6], pos, table, qw.cuda(), kw.cuda())  # noqa: E731
    (q, k), (q0, k0) = run(qkv.cuda()), run(clean.cuda())
    same_q, same_k = torch.ones(4, 4, dtype=torch.bool), torch.ones(4, 2, dtype=torch.bool)
    same_q[1, 2], same_k[2, 0] = False, False
    assert same_bits(q.cpu()[same_q], q0.cpu()[same_q]) and same_bits(k.cpu()[same_k], k0.cpu()[same_k])
    assert q[1, 2].isnan().any() and k[2, 0].isnan().all()


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 16, 1), (1, 8, 128, 16), (7, 2, 80, 3), (33, 8, 128, 16), (200, 16, 64, 128),
                                        (1023, 3, 256, 7), (2500, 8, 128, 64), (1700, 33, 32, 16), (5, 2, 96, 32), (5, 2, 48, 1)])
def test_store_gives_the_group_quantiser_s_codes(T, H, D, page, dtype):
    from sglang_b200.layers.quantization.kv_cache import store_kv_fp8
    qkv, _ = _inputs(T, 0, H, D, dtype, 7 * T + D)
    qkv[0, 0, 0], qkv[0, 0, 1], qkv[0, H, 3] = 300.0, -0.0, -1e-7
    pages = (2 * T + page - 1) // page + 1
    kc, vc, ks, vs = _cache(pages, page, H, D)
    before = [t.clone() for t in (kc, vc, ks, vs)]
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(T))[:T]
    slots[T // 3] = -1
    if T > 4:
        slots[T // 3 + 1], slots[T // 3 + 2] = pages * page, 1 << 40
    dev = qkv.cuda()
    store_kv_fp8(dev[:, :H], dev[:, H:], kc, vc, ks, vs, slots.cuda())
    ok = (slots >= 0) & (slots < pages * page)
    for x, cache, scale, old, old_s in ((qkv[:, :H], kc, ks, before[0], before[2]), (qkv[:, H:], vc, vs, before[1], before[3])):
        codes, s = O.quant_group_fp8_cuda_semantics(x.reshape(T, H * D), D)
        want, want_s = old.cpu().view(torch.uint8).flatten(0, 1), old_s.cpu().flatten(0, 1)
        want[slots[ok]] = codes.view(torch.uint8).view(T, H, D)[ok]
        want_s[slots[ok]] = s.view(T, H)[ok]
        assert torch.equal(cache.cpu().view(torch.uint8).flatten(0, 1), want)
        assert same_bits(scale.flatten(0, 1), want_s)


@pytest.mark.parametrize("T,H,D,page", [(40000, 1, 128, 16), (30011, 2, 64, 48), (20001, 3, 128, 64), (70003, 1, 32, 7), (9001, 5, 48, 1), (1500, 1, 112, 16),
                                        (12345, 2, 256, 16)])
def test_store_of_many_tokens_with_few_heads(T, H, D, page):
    """Rows of several tokens in one warp: the codes and scales are still the group quantiser's (heads of 32 and 48: those of a
    store of a few tokens at a time), skipped slots and the rest of the cache stay."""
    from sglang_b200.layers.quantization.kv_cache import store_kv_fp8
    g = torch.Generator().manual_seed(T)
    k, v = (torch.randn(T, H, D, generator=g).to(BF).cuda() for _ in range(2))
    pages = (T + 100 + page - 1) // page
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[::7] = -1
    slots[3] = pages * page
    def empty():
        return ([torch.zeros(pages, page, H, D, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
                + [torch.full((pages, page, H), 5.0, device="cuda") for _ in range(2)])
    got, want = empty(), empty()
    store_kv_fp8(k, v, *got, slots.cuda())
    for at in range(0, T, 1000):
        store_kv_fp8(k[at:at + 1000], v[at:at + 1000], *want, slots[at:at + 1000].cuda())
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    spare = torch.ones(pages * page, dtype=torch.bool)
    spare[slots[(slots >= 0) & (slots < pages * page)]] = False
    assert (got[2].cpu().view(-1, H)[spare] == 5).all() and (got[2].cpu().view(-1, H)[~spare] != 5).all()


def test_store_special_values_as_the_group_quantiser():
    """Infinities, NaN, zeros, the smallest numbers and a scale whose significand is all ones."""
    from sglang_b200.layers.quantization.kv_cache import store_kv_fp8
    x = torch.randn(8, 2, 64, generator=torch.Generator().manual_seed(1)).to(BF)
    x[0, 0], x[0, 1, 5], x[1, 0, 3], x[1, 1, 2] = 0.0, float("nan"), float("inf"), float("-inf")
    x[2, 0] = 1e-38
    x[2, 1] = torch.finfo(BF).max
    x[3, 0, :8] = torch.tensor([-0.0, 1e-30, -1e-30, 448.0, 2 ** -9, 2 ** -10, 3 * 2 ** -10, 447.0])
    kc, vc, ks, vs = _cache(2, 4, 2, 64)
    store_kv_fp8(x.cuda(), x.cuda(), kc, vc, ks, vs, torch.arange(8).int().cuda())
    codes, s = O.quant_group_fp8_cuda_semantics(x.view(8, 128), 64)
    for cache, scale in ((kc, ks), (vc, vs)):
        assert torch.equal(cache.cpu().view(torch.uint8).view(8, 128), codes.view(torch.uint8))
        assert same_bits(scale.view(8, 2), s)


def test_what_special_values_read_back_as():
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8, store_kv_fp8
    x = torch.ones(4, 1, 32, dtype=BF)
    x[0, 0, 3], x[0, 0, 4], x[1, 0, 5], x[2, 0, 6] = float("nan"), -3.5, float("inf"), float("-inf")
    x[3] = float("nan")
    cache = _cache(1, 4, 1, 32)
    store_kv_fp8(x.cuda(), x.cuda(), *cache, torch.arange(4).cuda())
    k, v = load_kv_fp8(*cache, torch.zeros(1, 1).int().cuda(), torch.tensor([0, 4]).int().cuda(), 4)
    for out in (k.cpu()[:, 0], v.cpu()[:, 0]):
        assert out[0, 3] == -3.5 and out[0, 4] == -3.5 and (out[0, 5:] == 1).all()
        for t, d in ((1, 5), (2, 6)):
            rest = torch.arange(32) != d
            assert out[t, d] == float("-inf") and out[t, rest].isnan().all()
        assert (out[3] == torch.tensor(-1e-10).to(BF)).all()


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,neox,page", [(1, 64, 8, 128, 128, True, 64), (1, 1, 1, 32, 16, False, 1),
                                                      (30, 10, 2, 96, 48, True, 5), (64, 8, 8, 64, 64, False, 16),
                                                      (900, 64, 8, 128, 128, True, 64), (130, 4, 1, 256, 128, True, 128)])
def test_fused_store(T, Hq, Hkv, D, rot, neox, page, dtype):
    from sglang_b200.layers.quantization.kv_cache import qk_norm_rope_store_kv_fp8
    from sglang_b200.layers.rotary_embedding import qk_norm_rope
    qkv, (qw, kw) = _inputs(T, Hq, Hkv, D, dtype, T + 3 * D)
    pos = torch.randint(0, 5000, (T,), generator=torch.Generator().manual_seed(T))
    pos[T // 2 + 1:T // 2 + 2] = -1                            # padding in the middle
    table = _table(5000, rot)
    pages = (2 * T + page - 1) // page + 1
    kc, vc, ks, vs = _cache(pages, page, Hkv, D)
    before = [t.clone() for t in (kc, vc, ks, vs)]
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(T))[:T]
    slots[T // 4:T // 4 + 1] = -1 if T > 1 else slots[0]
    dev = qkv.cuda()
    q, k, v = _split(dev, Hq, Hkv)
    args = (pos.cuda(), table.cuda(), kc, vc, ks, vs, slots.cuda(), qw.cuda(), kw.cuda())
    qo, ko = torch.zeros(T, Hq, D, dtype=dtype, device="cuda"), torch.zeros(T, Hkv, D, dtype=dtype, device="cuda")
    qk_norm_rope_store_kv_fp8(q, k, v, *args, is_neox=neox, q_out=qo, k_out=ko)
    qr, kr = qk_norm_rope(q, k, pos.cuda(), table.cuda(), qw.cuda(), kw.cuda(), is_neox=neox,
                          q_out=torch.zeros_like(qo), k_out=torch.zeros_like(ko))
    assert same_bits(qo, qr) and same_bits(ko, kr)
    ok = (slots >= 0) & (pos >= 0)
    # values: the group quantiser's bits; everything else in the cache as before
    codes, s = O.quant_group_fp8_cuda_semantics(qkv[:, Hq + Hkv:].reshape(T, Hkv * D), D)
    want, want_s = before[1].cpu().view(torch.uint8).flatten(0, 1), before[3].cpu().flatten(0, 1)
    want[slots[ok]], want_s[slots[ok]] = codes.view(torch.uint8).view(T, Hkv, D)[ok], s.view(T, Hkv)[ok]
    assert torch.equal(vc.cpu().view(torch.uint8).flatten(0, 1), want) and same_bits(vs.flatten(0, 1), want_s)
    others = torch.ones(pages * page, dtype=torch.bool)
    others[slots[ok]] = False
    assert torch.equal(kc.cpu().view(torch.uint8).flatten(0, 1)[others], before[0].cpu().view(torch.uint8).flatten(0, 1)[others])
    assert same_bits(ks.cpu().flatten(0, 1)[others], before[2].cpu().flatten(0, 1)[others])
    # keys: max(|y_a|, |y_b|) >= (|a cos| + |b sin|) / 2, so a scale is off by 2 steps relative to itself at most, each way;
    # a code by half a step of e4m3 (2^-4 of the value, or 2^-10 of the scale below its normal range)
    y, _ = _exact(qkv[:, Hq:Hq + Hkv], kw, pos.clamp_min(0), table, neox, 1e-6)
    y, amax = y[ok], y[ok].abs().amax(-1).clamp_min(1e-10)
    scale = ks.cpu().flatten(0, 1)[slots[ok]].double()
    slack = 4 * _steps(D) + 2 ** -23
    assert ((scale - amax / 448).abs() <= slack * amax / 448).all()
    back = kc.cpu().flatten(0, 1).float()[slots[ok]].double() * scale[..., None]
    assert ((back - y).abs() <= 2 ** -4 * y.abs() + 2 ** -10 * scale[..., None] + 2 * slack * amax[..., None]).all()
    # without k_out, q in place
    kc2, vc2, ks2, vs2 = before
    out = qk_norm_rope_store_kv_fp8(q, k, v, args[0], args[1], kc2, vc2, ks2, vs2, *args[6:], is_neox=neox, q_out=q)
    live = (pos >= 0).cuda()
    assert out.data_ptr() == q.data_ptr() and same_bits(q[live], qo[live])
    assert same_bits(kc2, kc) and same_bits(ks2, ks) and same_bits(vc2, vc) and same_bits(vs2, vs)
    assert same_bits(dev[:, Hq:], qkv[:, Hq:])


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D,neox", [(32, True), (64, False), (128, True), (256, False)])
def test_fused_keys_get_the_correctly_rounded_quotient(D, neox, dtype):
    """With no norm and sines of zero a key is fp32(x cos), which is known to the bit, and so are its codes and scale: also where the
    scale's significand is all ones (largest magnitudes just below 448 times a power of two), which no 16-bit number divided by
    448 gives and which the quotient by the reciprocal is not made for."""
    from sglang_b200.layers.quantization.kv_cache import qk_norm_rope_store_kv_fp8
    T, H = 64, 2
    g = torch.Generator().manual_seed(D)
    x = (torch.rand(T, H, D, generator=g) * 2 - 1).to(dtype)
    x[x == 0] = 0.5
    x[:, :, 5] = -1.0                                          # the largest magnitude of every row
    below = torch.tensor([448.0 * 2.0 ** -e for e in range(32)])
    cos = torch.cat([torch.nextafter(below, torch.zeros(32)), torch.rand(32, generator=g) * 3 + 0.1])
    table = torch.cat([cos[:, None].expand(T, D // 2), torch.zeros(T, D // 2)], 1).contiguous()
    y = x.float() * cos[:, None, None]                         # one fp32 product each, as in the kernel
    codes, s = O.quant_group_fp8_cuda_semantics(y.reshape(T, H * D), D)
    assert (s[:32].view(torch.int32) & 0x7fffff == 0x7fffff).all()
    kc, vc, ks, vs = _cache(4, 16, H, D)
    xd = x.cuda()
    qk_norm_rope_store_kv_fp8(xd[:, :1], xd, xd.clone(), torch.arange(T).cuda(), table.cuda(), kc, vc, ks, vs, torch.arange(T).cuda(), is_neox=neox)
    assert same_bits(ks.view(T, H), s)
    assert torch.equal(kc.cpu().view(torch.uint8).view(T, H * D), codes.view(torch.uint8))


def test_fused_store_of_a_position_outside_the_table_reads_as_nan():
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8, qk_norm_rope_store_kv_fp8
    qkv, (qw, kw) = _inputs(2, 4, 2, 64, BF, 11)
    kc, vc, ks, vs = _cache(2, 2, 2, 64)
    q, k, v = _split(qkv.cuda(), 4, 2)
    out = qk_norm_rope_store_kv_fp8(q, k, v, torch.tensor([3, 50]).cuda(), _table(50, 64).cuda(), kc, vc, ks, vs,
                                    torch.tensor([0, 1]).cuda(), qw.cuda(), kw.cuda())
    kl, vl = load_kv_fp8(kc, vc, ks, vs, torch.tensor([[0]]).int().cuda(), torch.tensor([0, 2]).int().cuda(), 2)
    assert out[1].isnan().all() and kl[1].isnan().all() and not (out[0].isnan().any() or kl[0].isnan().any() or vl.isnan().any())


def _paged(lens, page, starts=None, seed=0):
    """A page table for sequences that end after starts + lens tokens, and the slot of every token read."""
    g = torch.Generator().manual_seed(seed)
    starts = starts if starts is not None else [0] * len(lens)
    per = [(s + n + page - 1) // page for s, n in zip(starts, lens)]
    pages = sum(per) + 2
    ids = torch.randperm(pages, generator=g).int()
    table = torch.full((len(lens), max([1] + per)), -1, dtype=torch.int32)
    slots, at = [], 0
    for b, (s, n) in enumerate(zip(starts, lens)):
        table[b, :per[b]] = ids[at:at + per[b]]
        at += per[b]
        tok = torch.arange(s, s + n)
        slots.append(table[b, tok // page].long() * page + tok % page)
    indptr = torch.tensor([0] + list(lens)).cumsum(0).int()
    return pages, table, indptr, torch.cat(slots)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("lens,page,H,D", [([1], 16, 8, 128), ([0, 5, 0, 0, 17, 0], 4, 2, 64), ([100, 1, 203, 97], 16, 8, 128),
                                           ([33] * 70 + [0] * 70 + [2], 32, 1, 16), ([3000, 5, 1111], 64, 4, 256), ([7, 9], 1, 3, 80),
                                           ([1] * 1500, 8, 2, 32), ([0, 0, 0], 8, 2, 32),
                                           ([19000, 0, 37, 1], 16, 1, 16), ([9999, 12345], 64, 2, 48)])
def test_load(lens, page, H, D, dtype):
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8
    for starts in (None, [(5 * b) % 23 for b in range(len(lens))]):
        pages, table, indptr, slots = _paged(lens, page, starts)
        kc, vc, ks, vs = _cache(pages, page, H, D)
        n = int(indptr[-1])
        st = None if starts is None else torch.tensor(starts).int().cuda()
        k_out = torch.full((n + 5, H, D), 3.0, dtype=dtype, device="cuda")
        k, v = load_kv_fp8(kc, vc, ks, vs, table.cuda(), indptr.cuda(), n + 5, kv_start=st, out_dtype=dtype, k_out=k_out)
        assert k.data_ptr() == k_out.data_ptr() and (k[n:] == 3.0).all()
        for got, cache, scale in ((k, kc, ks), (v, vc, vs)):
            want = (cache.cpu().float().flatten(0, 1)[slots] * scale.cpu().flatten(0, 1)[slots][..., None]).to(dtype)
            assert same_bits(got[:n], want)


@pytest.mark.parametrize("n,H,D", [(1183, 1, 64), (1184, 1, 64), (2367, 1, 128), (2369, 1, 128), (4735, 2, 128), (4737, 2, 128), (9473, 4, 128),
                                   (18943, 8, 128), (18945, 8, 128), (5329, 3, 96)])
def test_load_on_both_sides_of_the_block_sizes(n, H, D):
    """Blocks of 8 rows and of 32, the larger from fewer tokens on where rows are short; the last one ends early."""
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8
    pages, table, indptr, slots = _paged([n // 3, 1, n - n // 3 - 1], 16)
    kc, vc, ks, vs = _cache(pages, 16, H, D)
    out = [torch.full((n + 40, H, D), 3.0, dtype=BF, device="cuda") for _ in range(2)]
    load_kv_fp8(kc, vc, ks, vs, table.cuda(), indptr.cuda(), n + 40, k_out=out[0], v_out=out[1])
    for got, cache, scale in ((out[0], kc, ks), (out[1], vc, vs)):
        want = (cache.cpu().float().flatten(0, 1)[slots] * scale.cpu().flatten(0, 1)[slots][..., None]).to(BF)
        assert same_bits(got[:n], want) and (got[n:] == 3.0).all()


def test_load_of_missing_pages_reads_as_nan():
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8
    pages, table, indptr, slots = _paged([20, 9], 4)
    table[0, 2], table[1, 0] = pages, -7
    kc, vc, ks, vs = _cache(pages, 4, 2, 64)
    long = torch.tensor([0, 25, 34]).int()                     # sequence 0 is longer than its row of the table
    k, v = load_kv_fp8(kc, vc, ks, vs, table.cuda(), long.cuda(), 34)
    bad = torch.zeros(34, dtype=torch.bool)
    bad[8:12] = bad[20:29] = True
    for t in (k, v):
        assert t.cpu()[bad].isnan().all() and not t.cpu()[~bad].isnan().any()


def test_load_through_a_table_without_columns():
    """No page of any sequence is in it: the rows of the sequences are NaN, those behind them stay."""
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8
    cache = _cache(2, 4, 2, 64)
    out = torch.full((5, 2, 64), 3.0, dtype=BF, device="cuda")
    k, v = load_kv_fp8(*cache, torch.empty(2, 0, dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 3]).int().cuda(), 5, k_out=out)
    assert k[:3].isnan().all() and v[:3].isnan().all() and (k[3:] == 3.0).all()


def test_permuted_and_sliced_caches():
    """[2, num_pages, num_kv_heads, page_size, head_dim] pools, passed as views."""
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8, store_kv_fp8
    pages, table, indptr, slots = _paged([37, 11], 8)
    H, D, n = 4, 96, 48
    qkv, _ = _inputs(n, 0, H, D, BF, 1)
    dev = qkv.cuda()
    plain = _cache(pages, 8, H, D)
    pool = torch.zeros(2, pages, H, 8, D, device="cuda").to(F8)
    scales = torch.zeros(pages, 2, 8, H, device="cuda")
    views = [pool[0].transpose(1, 2), pool[1].transpose(1, 2), scales[:, 0], scales[:, 1]]
    for c in (plain, views):
        store_kv_fp8(dev[:, :H], dev[:, H:], *c, slots.cuda())
    a = load_kv_fp8(*plain, table.cuda(), indptr.cuda(), n)
    wide = torch.zeros(n, 2 * H, D, dtype=BF, device="cuda")
    b = load_kv_fp8(*views, table.cuda(), indptr.cuda(), n, k_out=wide[:, :H], v_out=wide[:, H:])
    assert same_bits(a[0], b[0]) and same_bits(a[1], b[1])


def test_a_cache_beyond_32_bits():
    """Slots whose byte offset passes 2^32 (a 4.6 GB cache)."""
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8, store_kv_fp8
    H, D, page = 8, 128, 64
    pages = 70000
    kc = torch.empty(pages, page, H, D, dtype=F8, device="cuda")
    vc = kc                                                    # the values over the keys: the same data, so the same bytes
    ks = torch.empty(pages, page, H, device="cuda")
    x = torch.randn(5, H, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).to(BF)
    slots = torch.tensor([0, pages * page - 1, pages * page - 65, (1 << 32) // (H * D), (1 << 31) // (H * D)])
    store_kv_fp8(x, x, kc, vc, ks, ks, slots.cuda())
    table = (slots // page).int()[:, None]
    k, v = load_kv_fp8(kc, vc, ks, ks, table.cuda(), torch.arange(6).int().cuda(), 5, kv_start=(slots % page).int().cuda())
    codes, s = O.quant_group_fp8_cuda_semantics(x.cpu().view(5, H * D), D)
    want = (codes.float().view(5, H, D) * s.view(5, H, 1)).to(BF)
    assert same_bits(k, want) and same_bits(v, want)


def test_empty_calls():
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8, qk_norm_rope_store_kv_fp8, store_kv_fp8
    from sglang_b200.layers.rotary_embedding import qk_norm_rope
    z = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731
    cache = _cache(2, 4, 2, 64)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    q, k = qk_norm_rope(z(0, 4, 64), z(0, 2, 64), none, _table(8, 64).cuda())
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    store_kv_fp8(z(0, 2, 64), z(0, 2, 64), *cache, none)
    assert qk_norm_rope_store_kv_fp8(z(0, 4, 64), z(0, 2, 64), z(0, 2, 64), none, _table(8, 64).cuda(), *cache, none).shape == (0, 4, 64)
    k, v = load_kv_fp8(*cache, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), 0)
    assert k.shape == v.shape == (0, 2, 64)
