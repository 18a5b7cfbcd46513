"""CPU: what the adapter, head-norm and cache functions refuse, and the C ABI's codes for the same; nothing is launched."""
import ctypes

import pytest
import torch

BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _heads_call(**change):
    from sglang_b200.layers.rotary_embedding import qk_norm_rope
    a = dict(q=torch.zeros(3, 4, 64, dtype=BF), k=torch.zeros(3, 2, 64, dtype=BF), positions=torch.zeros(3, dtype=torch.int64),
             cos_sin_cache=torch.zeros(10, 64), q_weight=torch.ones(64, dtype=BF), k_weight=torch.ones(64, dtype=BF))
    a.update(change)
    return qk_norm_rope(**a)


@pytest.mark.parametrize("change,message", [
    ({}, "CUDA"),
    (dict(q=torch.zeros(3, 4, 64)), "bfloat16 or float16"),
    (dict(q=torch.zeros(3, 4, 64, dtype=F16)), "same type"),
    (dict(q=torch.zeros(3, 256, dtype=BF)), "q must be"),
    (dict(q=torch.zeros(2, 4, 64, dtype=BF)), "same number of tokens"),
    (dict(k=torch.zeros(3, 2, 40, dtype=BF)), "multiple of 16"),
    (dict(k=torch.zeros(3, 2, 272, dtype=BF)), "at most 256"),
    (dict(k=torch.zeros(3, 64, 2, dtype=BF).transpose(1, 2)), "last dimension"),
    (dict(k=torch.zeros(3, 2, 68, dtype=BF)[..., :64]), "multiples of 8"),
    (dict(k=torch.zeros(3 * 128 + 4, dtype=BF)[4:].view(3, 2, 64)), "aligned"),
    (dict(positions=None), "positions"),
    (dict(positions=torch.zeros(3)), "int32 or int64"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), "positions must have shape"),
    (dict(cos_sin_cache=torch.zeros(10, 64, dtype=BF)), "float32"),
    (dict(cos_sin_cache=torch.zeros(10, 24)), "rotary_dim"),
    (dict(cos_sin_cache=torch.zeros(10, 80)), "rotary_dim"),
    (dict(q_weight=torch.ones(32, dtype=BF)), "q_weight must have shape"),
    (dict(k_weight=torch.ones(64)), "k_weight must have the type"),
    (dict(q_out=torch.zeros(3, 4, 64, dtype=F16)), "q_out"),
    (dict(k_out=torch.zeros(3, 1, 64, dtype=BF).expand(3, 2, 64)), "expanded"),
    (dict(q="q"), "must be a tensor"),
])
def test_head_rows_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _heads_call(**change)


def _store_call(**change):
    from sglang_b200.layers.quantization.kv_cache import store_kv_fp8
    a = dict(k=torch.zeros(3, 2, 64, dtype=BF), v=torch.zeros(3, 2, 64, dtype=BF), k_cache=torch.zeros(5, 4, 2, 64).to(F8),
             v_cache=torch.zeros(5, 4, 2, 64).to(F8), k_scale=torch.zeros(5, 4, 2), v_scale=torch.zeros(5, 4, 2),
             slots=torch.zeros(3, dtype=torch.int32))
    a.update(change)
    return store_kv_fp8(**a)


@pytest.mark.parametrize("change,message", [
    ({}, "CUDA"),
    (dict(v=torch.zeros(3, 1, 64, dtype=BF)), "v must have shape"),
    (dict(v=torch.zeros(3, 2, 64, dtype=F16)), "same type"),
    (dict(v=None), "v must be given"),
    (dict(k_cache=torch.zeros(5, 4, 2, 64)), "float8_e4m3fn"),
    (dict(k_cache=torch.zeros(20, 2, 64).to(F8)), "k_cache must be"),
    (dict(v_cache=torch.zeros(5, 4, 2, 32).to(F8)), "v_cache must have shape"),
    (dict(k_scale=torch.zeros(5, 4, 2, dtype=BF)), "float32"),
    (dict(v_scale=torch.zeros(5, 4, 1)), "v_scale must have shape"),
    (dict(v_scale=torch.zeros(5, 4, 1).expand(5, 4, 2)), "expanded"),
    (dict(k=torch.zeros(3, 4, 64, dtype=BF), v=torch.zeros(3, 4, 64, dtype=BF)), "heads of k"),
    (dict(slots=torch.zeros(2, dtype=torch.int32)), "slots must have shape"),
    (dict(slots=torch.zeros(3)), "int32 or int64"),
    (dict(slots=torch.zeros(6, dtype=torch.int32)[::2]), "contiguous"),
])
def test_store_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _store_call(**change)


def _load_call(**change):
    from sglang_b200.layers.quantization.kv_cache import load_kv_fp8
    a = dict(k_cache=torch.zeros(5, 4, 2, 64).to(F8), v_cache=torch.zeros(5, 4, 2, 64).to(F8), k_scale=torch.zeros(5, 4, 2),
             v_scale=torch.zeros(5, 4, 2), page_table=torch.zeros(2, 3, dtype=torch.int32),
             kv_indptr=torch.zeros(3, dtype=torch.int32), num_tokens=7)
    a.update(change)
    return load_kv_fp8(**a)


@pytest.mark.parametrize("change,message", [
    ({}, "CUDA"),
    (dict(num_tokens=-1), "negative"),
    (dict(page_table=torch.zeros(2, 3, dtype=torch.int64)), "int32"),
    (dict(page_table=torch.zeros(2, 6, dtype=torch.int32)[:, ::2]), "last dimension"),
    (dict(kv_indptr=torch.zeros(2, dtype=torch.int32)), "kv_indptr must have shape"),
    (dict(kv_indptr=torch.zeros(3, dtype=torch.int64)), "int32"),
    (dict(kv_start=torch.zeros(3, dtype=torch.int32)), "kv_start must have shape"),
    (dict(out_dtype=torch.float32), "out_dtype"),
    (dict(k_out=torch.zeros(6, 2, 64, dtype=BF)), "k_out must have shape"),
    (dict(v_out=torch.zeros(7, 2, 64, dtype=F16)), "out_dtype"),
    (dict(k_cache=torch.zeros(5, 4, 2, 40).to(F8), v_cache=torch.zeros(5, 4, 2, 40).to(F8)), "multiple"),
])
def test_load_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _load_call(**change)


class _Batch:
    """What LoRABatch holds, without its launch."""

    def __init__(self, T, L):
        from sglang_b200 import _lib
        self.plan = torch.zeros(_lib.lib().b200_lora_plan_bytes(T, L), dtype=torch.uint8)
        self.num_adapters, self.scalings = L, torch.ones(L)


def _lora_call(**change):
    from sglang_b200.layers.lora import apply_lora
    a = dict(base_output=torch.zeros(5, 96, dtype=BF), x=torch.zeros(5, 64, dtype=BF), lora_a=torch.zeros(3, 32, 64, dtype=BF),
             lora_b=torch.zeros(3, 96, 16, dtype=BF), batch=_Batch(5, 3), output_sizes=[64, 32])
    a.update(change)
    return apply_lora(**a)


@pytest.mark.parametrize("change,message", [
    ({}, "CUDA"),
    (dict(x=torch.zeros(5, 64)), "type of x|bfloat16"),
    (dict(x=torch.zeros(1, 5, 64, dtype=BF)), "x must be"),
    (dict(x=torch.zeros(5, 72, dtype=BF)), "lora_a must be"),
    (dict(x=torch.zeros(5, 68, dtype=BF)[:, :64]), "multiples of 8"),
    (dict(lora_a=torch.zeros(3, 16, 64, dtype=BF)), "lora_a must be"),
    (dict(lora_a=torch.zeros(2, 32, 64, dtype=BF)), "adapters of the batch"),
    (dict(lora_a=torch.zeros(3, 32, 128, dtype=BF)[..., :64]), "contiguous"),
    (dict(lora_b=torch.zeros(3, 96, 16, dtype=F16)), "type of x"),
    (dict(lora_a=torch.zeros(3, 24, 64, dtype=BF), lora_b=torch.zeros(3, 96, 12, dtype=BF)), "R must be"),
    (dict(lora_a=torch.zeros(3, 528, 64, dtype=BF), lora_b=torch.zeros(3, 96, 264, dtype=BF)), "R must be"),
    (dict(output_sizes=[64, 24]), "add up"),
    (dict(output_sizes=[60, 36]), "multiples of 8"),
    (dict(output_sizes=[8] * 9), "slices"),
    (dict(base_output=torch.zeros(5, 88, dtype=BF)), "base_output must have shape"),
    (dict(base_output=torch.zeros(1, 96, dtype=BF).expand(5, 96)), "overlap"),
    (dict(out=torch.zeros(5, 96, dtype=F16)), "out must be"),
    (dict(batch=_Batch(6, 3)), "another number of tokens"),
])
def test_lora_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _lora_call(**change)


def test_lora_refuses_an_output_that_is_read_elsewhere():
    """Columns of one buffer beside one another are fine (they get as far as the question of the device)."""
    z = torch.zeros(5, 256, dtype=BF)
    for base, x, out, message in (
            (z[:, :96], z[:, 96:160], None, "CUDA"), (z[:, 160:], z[:, 96:160], z[:, :96], "CUDA"),
            (z[:, :96], z[:, 64:128], None, "no memory with x"), (z[:, 128:224], z[:, :64], z[:, 56:152], "no memory with x|base_output"),
            (z[:, :96], z[:, 192:], z[:, 8:104], "base_output itself"), (z[:1, :96].expand(5, 96), z[:, 192:], z[:, 96:192], "overlap"),
            (None, z[:, :64], z[:, :96], "no memory with x"),
            (None, z.view(10, 128)[:5, :64], z[:, 160:], "no memory with x")):
        with pytest.raises(RuntimeError, match=message):
            _lora_call(base_output=base, x=x, out=out)
    y = torch.zeros(10, 96, dtype=BF)
    with pytest.raises(RuntimeError, match="CUDA"):
        _lora_call(base_output=y[5:], out=y[:5])
    with pytest.raises(RuntimeError, match="base_output itself"):
        _lora_call(base_output=y[4:9], out=y[:5])


@pytest.mark.parametrize("stride", [0, 8])
def test_lora_refuses_rows_that_overlap(stride):
    """A row broadcast over all tokens would be read as if the rows followed one another."""
    from sglang_b200.layers.lora import lora_expand, lora_shrink
    x = torch.zeros(5, 64, dtype=BF).as_strided((5, 64), (stride, 1))
    with pytest.raises(RuntimeError, match="x must not overlap"):
        _lora_call(x=x)
    with pytest.raises(RuntimeError, match="x must not overlap"):
        lora_shrink(x, torch.zeros(3, 32, 64, dtype=BF), _Batch(5, 3), num_slices=2)
    h = torch.zeros(5, 32, dtype=BF).as_strided((5, 32), (stride, 1))
    with pytest.raises(RuntimeError, match="h must not overlap"):
        lora_expand(h, torch.zeros(3, 96, 16, dtype=BF), _Batch(5, 3), output_sizes=[64, 32])


@pytest.mark.parametrize("ids,ranks,message", [
    (torch.zeros(4, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), "token_adapters"),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(2), "lora_ranks"),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), "1024 adapters"),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(1025, dtype=torch.int32), "1024 adapters"),
    (torch.zeros(1, dtype=torch.int32).expand(1000001), torch.zeros(2, dtype=torch.int32), "contiguous"),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), "CUDA"),
])
def test_lora_batch_refusals(ids, ranks, message):
    from sglang_b200.layers.lora import LoRABatch
    with pytest.raises(RuntimeError, match=message):
        LoRABatch(ids, ranks, torch.ones(ranks.shape[0]))


def test_c_abi_codes():
    from sglang_b200 import _lib
    L, P = _lib.lib(), ctypes.c_void_p
    one, ref = P(16), ctypes.byref
    rows = _lib.Heads(16, 512, 64)
    cache = _lib.KVCache(16, 16, 16, 16, (512, 128, 64), (512, 128, 64), (8, 2, 1), (8, 2, 1), 5, 4)

    def nr(q=rows, k=rows, dt=2, pos=one, cs=one, rot=64, T=3, D=64, eps=1e-6):
        return L.b200_qk_norm_rope(ref(q), ref(k), ref(q), ref(k), dt, pos, 0, cs, 10, rot, 1, None, None, eps, T, 4, 2, D, None)
    assert nr(T=0) == 0
    assert nr(T=-1) == -3 and nr(D=40) == -3 and nr(rot=24) == -3 and nr(rot=80) == -3
    assert nr(D=272, rot=16) == -9 and nr(dt=0) == -2 and nr(pos=None) == -1
    assert nr(q=_lib.Heads(None, 512, 64)) == -1 and nr(q=_lib.Heads(8, 512, 64)) == -5 and nr(k=_lib.Heads(16, 516, 64)) == -5
    assert nr(q=_lib.Heads(16, -512, 64)) == -4 and nr(cs=P(8)) == -5

    def st(c=cache, v=ref(rows), slots=one, T=3):
        return L.b200_store_kv_fp8(ref(rows), v, 2, ref(c) if c else None, slots, 0, T, 2, 64, None)

    def changed(**kw):
        c = _lib.KVCache.from_buffer_copy(cache)
        for name, value in kw.items():
            setattr(c, name, value)
        return c
    assert st(c=None) == -1 and st(T=0) == 0 and st(v=None) == -1 and st(slots=None) == -1
    assert st(changed(page_size=0)) == -3 and st(changed(num_pages=1 << 29)) == -9 and st(changed(k=None)) == -1
    assert st(changed(v=8)) == -5 and st(changed(k_stride=(512, 128, 72))) == -5 and st(changed(v_scale_stride=(8, -2, 1))) == -4

    def ld(c=cache, table=one, T=7, batch=2, D=64, dt=2):
        return L.b200_load_kv_fp8(ref(c), table, 3, 3, one, None, batch, ref(rows), ref(rows), dt, T, 2, D, None)
    assert ld(T=0) == 0 and ld(batch=0) == 0 and ld(T=-1) == -3 and ld(D=24) == -3 and ld(dt=0) == -2 and ld(table=None) == -1
    assert ld(changed(num_pages=-1)) == -3

    plan = L.b200_lora_plan_bytes(5, 3)
    assert plan >= 16 + 4 * 5 and L.b200_lora_plan_bytes(-1, 3) == 0
    assert L.b200_lora_plan(one, 5, one, 0, one, plan, None) == -3
    assert L.b200_lora_plan(one, 5, one, 2000, one, plan, None) == -9
    assert L.b200_lora_plan(one, 5, one, 3, one, plan - 1, None) == -3
    assert L.b200_lora_plan(None, 5, one, 3, one, plan, None) == -1

    def sh(x=one, ld_=64, dt=2, T=5, K=64, R=16, S=2, hld=32, nbytes=plan):
        return L.b200_lora_shrink(x, ld_, one, dt, one, nbytes, T, 3, K, R, S, one, hld, None)
    assert sh(T=0) == 0 and sh(K=60) == -3 and sh(R=12) == -3 and sh(R=264) == -9 and sh(S=0) == -3 and sh(S=9, hld=144) == -9
    assert sh(dt=0) == -2 and sh(ld_=56) == -4 and sh(hld=24) == -4 and sh(x=None) == -1 and sh(x=P(8)) == -5 and sh(nbytes=0) == -3

    def ex(sizes=(64, 32), h=one, hld=32, old=96, bld=96, T=5):
        return L.b200_lora_expand(h, hld, one, 2, one, plan, one, T, 3, 16, (ctypes.c_int64 * len(sizes))(*sizes), len(sizes), one, bld,
                                  one, old, None)
    assert ex(T=0) == 0 and ex(sizes=(64, 36)) == -3 and ex(old=88) == -4 and ex(bld=88) == -4 and ex(hld=24) == -4
    assert ex(h=None) == -1 and ex(h=P(8)) == -5 and ex(sizes=(8,) * 9) == -9


@pytest.mark.parametrize("L", [1, 3, 10, 40, 1000])
def test_plans_of_different_batches_differ_in_size(L):
    """By its size a plan is told from one for another number of tokens, whose permutation lies elsewhere in it."""
    from sglang_b200 import _lib
    sizes = [_lib.lib().b200_lora_plan_bytes(T, L) for T in range(30000)]
    assert all(a < b for a, b in zip(sizes, sizes[1:]))


def test_lora_refuses_the_batch_of_fewer_tokens():
    """212 tokens of 3 adapters in tiles of 16 and 256 in tiles of 128."""
    from sglang_b200.layers.lora import lora_expand, lora_shrink
    x, out = torch.zeros(256, 64, dtype=BF), torch.zeros(256, 96, dtype=BF)
    with pytest.raises(RuntimeError, match="another number of tokens"):
        _lora_call(base_output=out, x=x, batch=_Batch(212, 3))
    with pytest.raises(RuntimeError, match="another number of tokens"):
        lora_shrink(x, torch.zeros(3, 32, 64, dtype=BF), _Batch(212, 3), num_slices=2)
    with pytest.raises(RuntimeError, match="another number of tokens"):
        lora_expand(x[:, :32].contiguous(), torch.zeros(3, 96, 16, dtype=BF), _Batch(212, 3), output_sizes=[64, 32])


def test_update_refuses_other_numbers_of_adapters_or_tokens(monkeypatch):
    """Two adapters and five for three tokens have plans of one size."""
    from types import SimpleNamespace

    from sglang_b200 import _lib
    from sglang_b200.layers import lora
    host, planned = _lib.host(), []

    def plan(ids, ranks, plan):
        planned.append(ranks.shape[0])
        return torch.zeros(_lib.lib().b200_lora_plan_bytes(ids.shape[0], ranks.shape[0]), dtype=torch.uint8)
    with monkeypatch.context() as m:
        m.setattr(lora._lib, "host", lambda: SimpleNamespace(lora_plan=plan))
        batch = lora.LoRABatch(torch.zeros(3, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.ones(2))
        batch.lora_ranks = torch.ones(5, dtype=torch.int32)
        with pytest.raises(RuntimeError, match="2 adapters, not 5"):
            batch.update()
        assert planned == [2]
    assert _lib.host() is host
    batch.lora_ranks, batch.token_adapters = torch.ones(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="plan must have shape"):
        batch.update()


@pytest.mark.parametrize("num_tokens", [0, 1, 5, 6, 11])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_tokens_behind_the_segments_have_no_adapter(monkeypatch, num_tokens, index):
    """A padded batch has more tokens than its requests, one cut short has fewer."""
    from types import SimpleNamespace

    from sglang_b200.layers import lora
    monkeypatch.setattr(lora._lib, "host", lambda: SimpleNamespace(lora_plan=lambda *a: None))
    ranks, scal = torch.ones(5, dtype=torch.int32), torch.ones(5)
    batch = lora.LoRABatch.from_segments(torch.tensor([4, -1, 0, 2], dtype=index), torch.tensor([2, 1, 0, 3], dtype=index), num_tokens, ranks, scal)
    want = torch.tensor(([4, 4, -1, 2, 2, 2] + [-1] * 5)[:num_tokens], dtype=torch.int32)
    assert batch.token_adapters.dtype == torch.int32 and torch.equal(batch.token_adapters, want)
    none = torch.zeros(0, dtype=index)
    assert torch.equal(lora.LoRABatch.from_segments(none, none, num_tokens, ranks, scal).token_adapters, torch.full((num_tokens,), -1, dtype=torch.int32))


def test_outputs_that_are_read_or_written_elsewhere_are_refused():
    """The heads of one qkv output beside one another are fine, also in place (such calls get as far as the question of the device)."""
    qkv, more = torch.zeros(3, 8, 64, dtype=BF), torch.zeros(3, 8, 64, dtype=BF)
    q, k = qkv[:, :4], qkv[:, 4:6]
    flat = torch.zeros(2000, dtype=BF)
    for change, message in (
            (dict(q=q, k=k), "CUDA"), (dict(q=q, k=k, q_out=q, k_out=k), "CUDA"), (dict(q=q, k=k, q_out=more[:, 2:6], k_out=more[:, :2]), "CUDA"),
            (dict(q=q, k=k, q_out=more[:, :4], k_out=more[:, 3:5]), "q_out must share no memory with k_out"),
            (dict(q=q, k=k, q_out=qkv[:, 2:6]), "q_out must share no memory with q or be it"),
            (dict(q=q, k=k, q_out=qkv[:, 4:]), "q_out must share no memory with k"), (dict(q=q, k=k, k_out=q[:, :2]), "k_out must share no memory with q"),
            (dict(q=q, k=k, q_out=q[[0]].expand(3, 4, 64)), "expanded"),
            (dict(q=q, k=k, q_out=flat.as_strided((3, 4, 64), (256, 48, 1))), "q_out must not overlap itself"),
            (dict(q=q, k=k, q_out=flat.as_strided((3, 4, 64), (128, 64, 1))), "q_out must not overlap itself"),
            (dict(q=q, k=k, q_out=flat.as_strided((3, 4, 64), (64, 192, 1))), "CUDA"),
            # heads and tokens in turn: every other run of 64
            (dict(q=q, k=flat.as_strided((3, 2, 64), (512, 128, 1)), k_out=flat.as_strided((3, 2, 64), (512, 128, 1), 64)), "CUDA"),
            (dict(q=q, k=flat.as_strided((3, 2, 64), (512, 128, 1)), k_out=flat.as_strided((3, 2, 64), (512, 128, 1), 56)), "k_out must share no memory with k"),
            # rows of another length, and tokens of one tensor in the gaps of the other
            (dict(q=q, k=flat.as_strided((3, 2, 64), (512, 128, 1)), k_out=flat.as_strided((3, 2, 64), (640, 64, 1), 256)), "CUDA"),
            (dict(q=q, k=flat.as_strided((3, 2, 64), (512, 128, 1)), k_out=flat.as_strided((3, 2, 64), (640, 64, 1), 192)), "CUDA"),
            (dict(q=q, k=flat.as_strided((3, 2, 64), (512, 128, 1)), k_out=flat.as_strided((3, 2, 64), (640, 64, 1), 128)), "k_out must share"),
            (dict(positions=more.view(torch.int64).view(-1)[:3], q=more[:, :4].clone(), k_out=more[:, :2]), "k_out must share no memory with positions"),
            (dict(q_weight=more[0, 1], k_out=more[:, :2]), "k_out must share no memory with q_weight")):
        with pytest.raises(RuntimeError, match=message):
            _heads_call(**change)


def test_caches_that_overlap_are_refused():
    """A pool that holds keys, values and scales in turn is fine."""
    k, v = torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, 2, 64, dtype=BF)
    pool, scales = torch.zeros(5, 2, 4, 2, 64).to(F8), torch.zeros(5, 4, 2, 2)
    page = torch.zeros(5, 2 * 4 * 2 * 68, dtype=torch.uint8)          # of keys, values and their scales, for each page
    codes = [page[:, i * 512:(i + 1) * 512].view(F8).view(5, 4, 2, 64) for i in range(2)]
    fp32 = [page[:, 1024 + i * 32:1056 + i * 32].view(torch.float32).view(5, 4, 2) for i in range(2)]
    both = dict(k_cache=pool[:, 0], v_cache=pool[:, 1], k_scale=scales[..., 0], v_scale=scales[..., 1])
    one = dict(both, v_cache=pool[:, 0], v_scale=scales[..., 0])
    for change, message in (
            (both, "CUDA"), (dict(k_cache=codes[0], v_cache=codes[1], k_scale=fp32[0], v_scale=fp32[1]), "CUDA"), (dict(one, v=k, k=k), "CUDA"),
            (one, "k_cache must share no memory with v_cache"),
            (dict(both, v_cache=pool.view(10, 4, 2, 64)[1:6]), "k_cache must share no memory with v_cache"),
            (dict(both, v_scale=scales[..., 0]), "k_scale must share no memory with v_scale"),
            (dict(both, k_scale=page[:, :32].view(torch.float32).view(5, 4, 2), k_cache=codes[0]), "k_cache must share no memory with k_scale"),
            (dict(both, k_cache=pool.view(-1).as_strided((5, 4, 2, 64), (512, 64, 64, 1))), "k_cache must not overlap itself"),
            (dict(both, slots=scales.view(torch.int32).view(-1)[:3]), "k_scale must share no memory with slots"),
            (dict(both, k=pool.view(-1).view(BF)[:384].view(3, 2, 64)), "k_cache must share no memory with k")):
        with pytest.raises(RuntimeError, match=message):
            _store_call(**dict(dict(k=k, v=v), **change))
    from sglang_b200.layers.quantization.kv_cache import qk_norm_rope_store_kv_fp8
    args = (k, k, k, torch.zeros(3, dtype=torch.int64), None)
    with pytest.raises(RuntimeError, match="k_cache must share no memory with v_cache"):      # the keys of a padded token are left out; values, too
        qk_norm_rope_store_kv_fp8(*args, *one.values(), torch.zeros(3, dtype=torch.int32))
    out = torch.zeros(7, 4, 64, dtype=BF)
    for change, message in ((dict(k_out=out[:, :2], v_out=out[:, 2:]), "CUDA"), (dict(k_out=out[:, :2], v_out=out[:, 1:3]), "k_out must share no memory with v_out"),
                            (dict(v_out=out.view(-1)[:1280].as_strided((7, 2, 64), (128, 48, 1))), "v_out must not overlap itself"),
                            (dict(k_out=torch.zeros(7, 2, 64, dtype=BF), kv_indptr=out.view(torch.int32).view(-1)[:3], v_out=out[:, :2]), "kv_indptr")):
        with pytest.raises(RuntimeError, match=message):
            _load_call(**change)


def test_memory_is_compared_byte_for_byte():
    """Random views of one buffer as output and input of a call: refused exactly when they share an element."""
    import random
    rng, buf = random.Random(0), torch.zeros(4000, dtype=BF)
    seen = [0, 0]
    for _ in range(3000):
        T, H = rng.randint(1, 4), rng.randint(1, 3)
        strides = [(rng.choice([32, 64, 96, 128, 256]), rng.choice([16, 32, 48, 64, 512])) for _ in range(2)]
        at = [8 * rng.randint(0, 60) for _ in range(2)]
        k, out = (buf.as_strided((T, H, 16), (*s, 1), o) for s, o in zip(strides, at))
        places = [torch.arange(4000).as_strided((T, H, 16), (*s, 1), o).flatten() for s, o in zip(strides, at)]
        if len(places[1].unique()) < places[1].numel():
            continue
        meets = bool(torch.isin(places[0], places[1]).any())
        with pytest.raises(RuntimeError) as e:
            _heads_call(q=torch.zeros(T, 1, 16, dtype=BF), k=k, k_out=out, positions=torch.zeros(T, dtype=torch.int64), cos_sin_cache=None,
                        q_weight=None, k_weight=None)
        if "overlap itself" in str(e.value):       # dimensions that interlock
            continue
        in_place = at[0] == at[1] and (T == 1 or strides[0][0] == strides[1][0]) and (H == 1 or strides[0][1] == strides[1][1])
        seen[meets] += 1
        assert ("CUDA" in str(e.value)) == (not meets or in_place), (T, H, strides, at, str(e.value))
    assert min(seen) > 300
