"""GPU: what stands between a decoder layer's normed input and its attention kernel, run together: the block-FP8 qkv
projection, the adapters of a mixed batch, head norms with the rotation, the cache written and read back."""
import pytest
import torch

from helpers import same_bits
from oracle import block_fp8_oracle as O

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HQ, HKV, D, K, R, L, PAGE = 8, 2, 128, 512, 16, 3, 16
SIZES = [HQ * D, HKV * D, HKV * D]


def _model():
    from sglang_b200.layers.quantization.fp8 import Fp8Config, Fp8LinearMethod
    method = Fp8LinearMethod(Fp8Config(is_checkpoint_fp8_serialized=True, weight_block_size=[128, 128]))
    layer = torch.nn.Module()
    method.create_weights(layer, K, SIZES, K, sum(SIZES), BF, device="cuda")
    wq, ws = O.gen_weight(sum(SIZES), K, seed=4)
    layer.weight.data.copy_(wq)
    layer.weight_scale_inv.data.copy_(ws)
    method.process_weights_after_loading(layer)
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).to(BF)  # noqa: E731
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    angle = torch.arange(512, dtype=torch.float64)[:, None] * inv
    return dict(method=method, layer=layer, A=rnd(L, 3 * R, K, scale=K ** -0.5), B=rnd(L, sum(SIZES), R, scale=0.1),
                ranks=torch.tensor([16, 8, 5], dtype=torch.int32, device="cuda"), scal=torch.tensor([1.0, 2.0, 0.5], device="cuda"),
                qw=1 + rnd(D, scale=0.1), kw=1 + rnd(D, scale=0.1), table=torch.cat([angle.cos(), angle.sin()], 1).float().cuda())


def _step(m, st):
    from sglang_b200.layers.lora import apply_lora
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8, qk_norm_rope_store_kv_fp8
    qkv = m["method"].apply(m["layer"], st["x"])
    base = qkv.clone()
    apply_lora(qkv, st["x"], m["A"], m["B"], st["batch"], output_sizes=SIZES)
    heads = qkv.view(-1, HQ + 2 * HKV, D)
    q = qk_norm_rope_store_kv_fp8(heads[:, :HQ], heads[:, HQ:HQ + HKV], heads[:, HQ + HKV:], st["pos"], m["table"], *st["cache"],
                                  st["slots"], m["qw"], m["kw"])
    k, v = load_kv_fp8(*st["cache"], st["pages"], st["indptr"], st["total"])
    return base, qkv, q, k, v


def _check(m, st, base, qkv, q, k, v, lens):
    """Each stage against its formula in 64 bits, from what the stage before gave."""
    c = lambda t: t.cpu().double()  # noqa: E731
    want = c(base)
    for t, a in enumerate(st["ids"].tolist()):
        if a < 0:
            continue
        r, at = int(m["ranks"][a]), 0
        for s, n in enumerate(SIZES):
            h = c(m["A"])[a, s * R:s * R + r] @ c(st["x"])[t]
            want[t, at:at + n] += float(m["scal"][a]) * c(m["B"])[a, at:at + n, :r] @ h
            at += n
    # bf16: half a step of the result, and half a step of h through the sum over r
    part = (want - c(base)).abs().amax()
    assert ((c(qkv) - want).abs() <= 2 ** -8 * want.abs() + 2 ** -8 * 4 * part).all()
    heads, pos = c(qkv).view(-1, HQ + 2 * HKV, D), st["pos"].cpu()

    def turned(x, w):
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * c(w)
        cs, sn = (p[:, None] for p in c(m["table"])[pos].chunk(2, dim=1))
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * cs - b * sn, b * cs + a * sn], dim=-1)
    y = turned(heads[:, :HQ], m["qw"])
    assert ((c(q) - y).abs() <= 2 ** -8 * y.abs() + 2 ** -16 * y.abs().amax()).all()
    # the new tokens, read back: half a step of e4m3 and half a step of bf16
    new, at = [], 0
    for n, cached in zip(lens, st["indptr"].diff().tolist()):
        new += list(range(at + cached - n, at + cached))
        at += cached
    for got, x in ((k, turned(heads[:, HQ:HQ + HKV], m["kw"])), (v, heads[:, HQ + HKV:])):
        amax = x.abs().amax(-1, keepdim=True)
        assert ((c(got)[new] - x).abs() <= (2 ** -4 + 2 ** -7) * x.abs() + (2 ** -10 / 448 + 2 ** -16) * amax).all()


def _batch(m, lens, cached, ids, seed):
    """Requests that have `cached` tokens in the cache and bring lens new ones."""
    from sglang_b200.layers.lora import LoRABatch
    g = torch.Generator().manual_seed(seed)
    total = [a + b for a, b in zip(cached, lens)]
    per = [(n + PAGE - 1) // PAGE for n in total]
    perm, at = torch.randperm(sum(per), generator=g).int(), 0
    pages = torch.full((len(lens), max(per)), -1, dtype=torch.int32)
    slots, pos = [], []
    for b, n in enumerate(per):
        pages[b, :n] = perm[at:at + n]
        at += n
        tok = torch.arange(cached[b], total[b])
        pos.append(tok)
        slots.append(pages[b, tok // PAGE].long() * PAGE + tok % PAGE)
    token_ids = torch.repeat_interleave(torch.tensor(ids), torch.tensor(lens)).int()
    st = dict(x=torch.randn(sum(lens), K, generator=g).to(BF).cuda(), pos=torch.cat(pos).cuda(), slots=torch.cat(slots).cuda(),
              pages=pages.cuda(), indptr=torch.tensor([0] + total).cumsum(0).int().cuda(), total=sum(total), ids=token_ids.cuda())
    st["batch"] = LoRABatch(st["ids"], m["ranks"], m["scal"])
    gc = torch.Generator(device="cuda").manual_seed(seed)
    codes = lambda: torch.randn(sum(per), PAGE, HKV, D, generator=gc, device="cuda").to(torch.float8_e4m3fn)  # noqa: E731
    st["cache"] = [codes(), codes(), torch.rand(sum(per), PAGE, HKV, generator=gc, device="cuda"),
                   torch.rand(sum(per), PAGE, HKV, generator=gc, device="cuda")]
    return st


@pytest.mark.parametrize("lens,cached,ids", [([1, 1, 1, 1], [0, 15, 16, 200], [0, 2, -1, 0]), ([70, 1, 33], [0, 64, 5], [1, 0, -1])])
def test_together(lens, cached, ids):
    m = _model()
    st = _batch(m, lens, cached, ids, 3)
    before = [t.clone() for t in st["cache"]]
    eager = _step(m, st)
    _check(m, st, *eager, lens)
    # the same step captured, replayed after the cache has been put back: the same bits
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = _step(m, st)
    for t, old in zip(st["cache"], before):
        t.copy_(old)
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(eager, captured):
        assert same_bits(a, b)


def test_what_is_written_in_place_counts_as_modified():
    """Autograd refuses to go back through what it kept of a tensor that a call has overwritten; tensors of inference mode, which have
    no such count, are written all the same."""
    from sglang_b200.layers.lora import LoRABatch, apply_lora
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8, qk_norm_rope_store_kv_fp8, store_kv_fp8
    from sglang_b200.layers.rotary_embedding import qk_norm_rope
    T = 3

    def run():
        ids = torch.zeros(T, dtype=torch.int32, device="cuda")
        z = lambda *s: torch.randn(*s, device="cuda").to(BF)  # noqa: E731
        batch = LoRABatch(ids, torch.full((1,), 8, dtype=torch.int32, device="cuda"), torch.ones(1, device="cuda"))
        base, x, A, B, q, k, v, w = z(T, 64), z(T, 128), z(1, 8, 128), z(1, 64, 8), z(T, 2, 64), z(T, 1, 64), z(T, 1, 64), z(64)
        caches = [torch.zeros(1, 4, 1, 64, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
        caches += [torch.zeros(1, 4, 1, device="cuda") for _ in range(2)]
        slots, ko, vo = torch.arange(T, device="cuda"), z(T, 1, 64), z(T, 1, 64)
        out = torch.empty_like(base)
        return ((lambda: batch.update(), [batch.plan], [ids]), (lambda: apply_lora(base, x, A, B, batch), [base], [x, A, B]),
                (lambda: apply_lora(base, x, A, B, batch, out=out), [out], [base, x]), (lambda: qk_norm_rope(q, k, None, None, w, w, q_out=q, k_out=k), [q, k], [w]),
                (lambda: store_kv_fp8(k, v, *caches, slots), caches, [k, v, slots]),
                (lambda: qk_norm_rope_store_kv_fp8(q, k, v, None, None, *caches, slots, w, w, q_out=q), caches + [q], [k, v]),
                (lambda: load_kv_fp8(*caches, ids[:1, None], slots[:2].int(), T, k_out=ko, v_out=vo), [ko, vo], caches))
    for call, written, read in run():
        before = [t._version for t in written], [t._version for t in read]
        call()
        assert all(t._version > n for t, n in zip(written, before[0])) and [t._version for t in read] == before[1]
    with torch.inference_mode():
        calls = run()
    for call, _, _ in calls:
        call()
    leaf = torch.randn(T, 64, device="cuda", dtype=BF, requires_grad=True)
    base = leaf * 1
    kept = base.exp().sum() + (base * base).sum()
    ids = torch.zeros(T, dtype=torch.int32, device="cuda")
    batch = LoRABatch(ids, torch.full((1,), 8, dtype=torch.int32, device="cuda"), torch.ones(1, device="cuda"))
    with torch.no_grad():
        apply_lora(base, torch.ones(T, 128, device="cuda", dtype=BF), torch.ones(1, 8, 128, device="cuda", dtype=BF),
                   torch.ones(1, 64, 8, device="cuda", dtype=BF), batch)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
