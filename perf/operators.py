"""What an attention layer does between its projections and its attention kernel, as timed cases:

  lora       low-rank adapters of many requests beside one shared projection: out = base + scaling * (x A^T) B^T, each token
             with the A and B of its own adapter (or none), the projection's output in one to three slices
  norm_rope  RMSNorm of every query and key head and the rotary position embedding, one pass
  fused      the same, and keys and values quantised to e4m3 (one fp32 scale for each token and head) into a paged cache
  store      keys and values quantised into the paged cache as they are
  load       a paged e4m3 cache read back as 16-bit keys and values, the sequences packed one behind the other

Projection sizes are those of the benchmark configurations; 64 query heads over 8 key/value heads of 128 are the
heads of the qkv projection with K = 8192, N = 10240.
"""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FP8 = torch.float8_e4m3fn
POSITIONS = 32768      # rows of the table of cosines and sines
EPS = 1e-6             # of the head norms


def listed():
    return [
        # one request with a rank-16 adapter decodes through the o projection: two small weight reads, latency
        {"name": "lora_1_o_proj", "kind": "lora", "dtype": "bf16", "T": 1, "K": 8192, "sizes": "8192", "R": 16, "L": 4,
         "segments": 1, "bare": 0.0},
        # a decode batch in which 32 adapters of several ranks are mixed and some requests have none: qkv projection
        {"name": "lora_128_qkv_mixed", "kind": "lora", "dtype": "bf16", "T": 128, "K": 8192, "sizes": "8192,1024,1024",
         "R": 64, "L": 32, "segments": 128, "bare": 0.125},
        # a prefill of 13 prompts with 8 adapters, an odd number of tokens in all, through the qkv projection, fp16
        {"name": "lora_8191_qkv", "kind": "lora", "dtype": "fp16", "T": 8191, "K": 8192, "sizes": "8192,1024,1024", "R": 64,
         "L": 8, "segments": 13, "bare": 0.0},
        # a prefill through gate_up, the widest output
        {"name": "lora_4096_gate_up", "kind": "lora", "dtype": "bf16", "T": 4096, "K": 7168, "sizes": "18432,18432", "R": 32,
         "L": 4, "segments": 5, "bare": 0.05},
        # a decode batch of 16
        {"name": "norm_rope_16", "kind": "norm_rope", "dtype": "bf16", "T": 16, "Hq": 64, "Hkv": 8, "D": 128, "rot": 128,
         "neox": True, "norm": True, "segments": 16},
        # prefill, pairs of neighbouring elements rotated, half of each head
        {"name": "norm_rope_8192_half", "kind": "norm_rope", "dtype": "fp16", "T": 8192, "Hq": 32, "Hkv": 4, "D": 128,
         "rot": 64, "neox": False, "norm": True, "segments": 7},
        # a decode batch of 64 writes its tokens into the cache
        {"name": "fused_64", "kind": "fused", "dtype": "bf16", "T": 64, "Hq": 64, "Hkv": 8, "D": 128, "rot": 128,
         "neox": True, "norm": True, "segments": 64, "page": 64},
        # a prefill of 8192 tokens writes its tokens into the cache
        {"name": "fused_8192", "kind": "fused", "dtype": "bf16", "T": 8192, "Hq": 64, "Hkv": 8, "D": 128, "rot": 128,
         "neox": True, "norm": True, "segments": 5, "page": 64},
        # keys that another kernel has rotated: a decode batch with an odd size
        {"name": "store_33", "kind": "store", "dtype": "bf16", "T": 33, "Hkv": 8, "D": 128, "segments": 33, "page": 16},
        # and a prefill, small heads
        {"name": "store_16384_d64", "kind": "store", "dtype": "fp16", "T": 16384, "Hkv": 16, "D": 64, "segments": 9, "page": 128},
        # the cached prefix of a few short requests
        {"name": "load_4x100", "kind": "load", "dtype": "bf16", "T": 401, "Hkv": 8, "D": 128, "segments": 4, "page": 16},
        # the prefixes of 37 long requests ahead of a chunk of prefill
        {"name": "load_37x3500", "kind": "load", "dtype": "bf16", "T": 131001, "Hkv": 8, "D": 128, "segments": 37, "page": 64},
    ]


def _log(rng, lo, hi):
    return min(hi, int(lo * (hi / lo) ** rng.random() + 0.5))


def draw(rng):
    kind = rng.choice(["lora", "norm_rope", "fused", "store", "load"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "lora":
        K, sizes = rng.choice([(7168, "18432,18432"), (18432, "7168"), (7168, "4096"), (7168, "576"), (8192, "8192,1024,1024"),
                               (8192, "8192"), (8192, "1024,128,128"), (1024, "8192"), (3584, "8192"), (4096, "8192"),
                               (8192, "3584,3584")])
        R, L = rng.choice([8, 16, 32, 40, 64]), _log(rng, 1, 32)
        N, slices = sum(map(int, sizes.split(","))), sizes.count(",") + 1
        T = _log(rng, 1, min(16384, 4096 * 36864 // N, 8191 * 8192 * 1536 // (K * L * R * slices), 8191 * 10240 * 512 // (N * L * R)))
        segments = T if T <= 256 else _log(rng, 1, 32)
        return {"kind": kind, "dtype": dtype, "T": T, "K": K, "sizes": sizes, "R": R, "L": L, "segments": segments,
                "bare": rng.choice([0.0, 0.05, 0.3])}
    Hkv, D, page = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 96, 128, 192, 256]), rng.choice([1, 16, 32, 64, 128])
    if kind == "load":
        T = _log(rng, 1, 131001 * 1024 // (Hkv * D))
        return {"kind": kind, "dtype": dtype, "T": min(T, 200000), "Hkv": Hkv, "D": D, "segments": _log(rng, 1, 256), "page": page}
    T = _log(rng, 1, 16384)
    segments = T if T <= 256 else _log(rng, 1, 32)
    if kind == "store":
        return {"kind": kind, "dtype": dtype, "T": T, "Hkv": Hkv, "D": D, "segments": segments, "page": page}
    Hq = Hkv * rng.choice([1, 4, 5, 8])
    case = {"kind": kind, "dtype": dtype, "T": min(T, 8192 * 10240 // ((Hq + 2 * Hkv) * D)), "Hq": Hq, "Hkv": Hkv, "D": D,
            "rot": rng.choice([D, D // 2]), "neox": rng.random() < 0.7, "norm": rng.random() < 0.8}
    case["segments"] = min(segments, case["T"])
    return dict(case, page=page) if kind == "fused" else case


# ------------------------------------------------------------------------------------------------------- inputs
def _lengths(case, g):
    """`segments` lengths that add up to T, ragged; every one at least 1 while there are as many tokens."""
    T, n = case["T"], case["segments"]
    cuts = torch.randperm(T - 1, generator=g)[:max(0, min(n, T) - 1)].sort().values + 1
    ends = torch.cat([cuts, torch.tensor([T])])
    lens = torch.diff(ends, prepend=torch.tensor([0]))
    return torch.cat([lens, lens.new_zeros(n - lens.numel())])


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _positions(lens, g):
    """Where each token stands in its request: a request of one token anywhere, longer ones behind a cached prefix."""
    T = int(lens.sum())
    begin = (torch.rand(lens.numel(), generator=g) * (POSITIONS - lens)).to(torch.int64)
    first = torch.cumsum(lens, 0) - lens
    return (torch.arange(T) + torch.repeat_interleave(begin - first, lens)).to("cuda")


def _cos_sin(rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _heads(case, gc, dt, heads):
    """The output of a qkv projection [T, heads * D] seen as heads: some heads larger than others, a few outliers."""
    T, D = case["T"], case["D"]
    x = _randn(gc, T, heads, D)
    x *= torch.exp2(_randn(gc, heads, 1))
    x[torch.rand(T, heads, D, generator=gc, device="cuda") < 1e-3] *= 20
    return x.to(dt)


def _cache(case, pages, gc):
    """A cache that holds other tokens already."""
    shape = (pages, case["page"], case["Hkv"])
    made = {}
    for name in ("k", "v"):
        made[name + "_cache"] = _randn(gc, *shape, case["D"], scale=100.0).clamp(-448, 448).to(FP8)
        made[name + "_scale"] = torch.rand(*shape, generator=gc, device="cuda") * 0.02 + 1e-3
    return made


def prepare(case, seed):
    g, gc = torch.Generator().manual_seed(seed), torch.Generator(device="cuda").manual_seed(seed)
    dt, T, kind = DTYPES[case["dtype"]], case["T"], case["kind"]
    lens = _lengths(case, g)
    s = {"kind": kind}
    if kind == "lora":
        K, R, L, sizes = case["K"], case["R"], case["L"], [int(n) for n in case["sizes"].split(",")]
        S, N = len(sizes), sum(sizes)
        # adapters dealt to the requests in turn, some requests without one; ranks R, R / 2 and R / 4
        ids = torch.arange(lens.numel()) % L
        ids[torch.rand(lens.numel(), generator=g) < case["bare"]] = -1
        ranks = torch.tensor([max(1, R >> (a % 3)) for a in range(L)], dtype=torch.int32)
        inside = (torch.arange(R)[None] < ranks[:, None]).to("cuda")
        s.update(sizes=sizes, x=_randn(gc, T, K, dtype=dt), base=_randn(gc, T, N, dtype=dt), out=torch.empty(T, N, dtype=dt, device="cuda"),
                 lora_a=(_randn(gc, L, S, R, K, scale=K ** -0.5) * inside[:, None, :, None]).to(dt).view(L, S * R, K),
                 lora_b=(_randn(gc, L, N, R, scale=0.05) * inside[:, None, :]).to(dt),
                 ids=torch.repeat_interleave(ids, lens).to(torch.int32).to("cuda"), ranks=ranks.to("cuda"),
                 scalings=(torch.rand(L, generator=g) * 1.5 + 0.5).to("cuda"))
        if own:
            from sglang_b200.layers.lora import LoRABatch
            # made once for a batch of tokens and used by every projection of every layer
            s["batch"] = LoRABatch(s["ids"], s["ranks"], s["scalings"])
        return s
    Hkv, D = case["Hkv"], case["D"]
    if kind == "load":
        page = case["page"]
        per = (lens + page - 1) // page
        pages = int(per.sum()) + 7
        s.update(_cache(case, pages, gc))
        table = torch.full((lens.numel(), max(1, int(per.max()))), -1, dtype=torch.int32)
        table[torch.arange(table.shape[1])[None] < per[:, None]] = torch.randperm(pages, generator=g)[:pages - 7].to(torch.int32)
        indptr = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(lens, 0)]).to(torch.int32)
        s.update(page_table=table.to("cuda"), indptr=indptr.to("cuda"), tokens=T, dtype=dt)
        return s
    if kind in ("fused", "store"):
        pages = (3 * T // 2 + case["page"] - 1) // case["page"] + 3
        s.update(_cache(case, pages, gc))
        s["slots"] = torch.randperm(pages * case["page"], generator=gc, device="cuda")[:T].sort().values
    if kind == "store":
        kv = _heads(case, gc, dt, 2 * Hkv)
        s.update(k=kv[:, :Hkv], v=kv[:, Hkv:])
        return s
    Hq = case["Hq"]
    qkv = _heads(case, gc, dt, Hq + 2 * Hkv)
    s.update(q=qkv[:, :Hq], k=qkv[:, Hq:Hq + Hkv], v=qkv[:, Hq + Hkv:], positions=_positions(lens, g),
             cos_sin=_cos_sin(case["rot"]), neox=case["neox"], q_weight=None, k_weight=None)
    if case["norm"]:
        s.update(q_weight=(1 + _randn(gc, D, scale=0.2)).to(dt), k_weight=(1 + _randn(gc, D, scale=0.2)).to(dt))
    return s


# ------------------------------------------------------------------------------------------------------- one pass
def _plain_lora(s):
    x, A, B, ids = s["x"], s["lora_a"], s["lora_b"], s["ids"]
    L, N, R = B.shape
    S = len(s["sizes"])
    h = (x.float() @ A.float().view(L * S * R, -1).T).view(-1, L, S, R)
    mine = (ids[:, None] == torch.arange(L, device=x.device))[:, :, None] & (torch.arange(R, device=x.device) < s["ranks"][:, None])
    h = torch.where(mine[:, :, None, :], h * s["scalings"][:, None, None], 0.0)
    b = B.float().transpose(1, 2).split(s["sizes"], dim=2)
    delta = torch.cat([h[:, :, i].flatten(1) @ b[i].flatten(0, 1) for i in range(S)], dim=1)
    return (s["base"].float() + delta).to(x.dtype)


def _plain_rows(x, weight, c, sn, neox):
    """fp32 heads x [T, H, D], normalised when there is a weight, their first 2 * c.shape[1] elements rotated."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    half = c.shape[1]
    c, sn = c[:, None], sn[:, None]
    if neox:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * sn, b * c + a * sn], dim=-1)
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * sn, b * c + a * sn], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _plain_norm_rope(s):
    c, sn = s["cos_sin"][s["positions"]].chunk(2, dim=1)
    return _plain_rows(s["q"], s["q_weight"], c, sn, s["neox"]), _plain_rows(s["k"], s["k_weight"], c, sn, s["neox"])


def _plain_store(s, name, x):
    x = x.float()
    scale = x.abs().amax(-1).clamp_min(1e-10) / 448.0
    codes = (x / scale[..., None]).clamp(-448, 448).to(FP8)
    s[name + "_cache"].view(torch.uint8).flatten(0, 1)[s["slots"]] = codes.view(torch.uint8)
    s[name + "_scale"].flatten(0, 1)[s["slots"]] = scale
    return s[name + "_cache"], s[name + "_scale"]


def _plain_load(s):
    page = s["k_cache"].shape[1]
    row = torch.arange(s["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["indptr"][1:], row, right=True)
    at = (row - s["indptr"][seq]).long()
    slot = s["page_table"][seq, at // page].long() * page + at % page
    both = [(s[n + "_cache"].view(torch.uint8).flatten(0, 1)[slot].view(FP8).float()
             * s[n + "_scale"].flatten(0, 1)[slot][..., None]).to(s["dtype"]) for n in ("k", "v")]
    return both[0], both[1]


def run(s):
    kind = s["kind"]
    if not own:
        if kind == "lora":
            return _plain_lora(s)
        if kind == "norm_rope":
            q, k = _plain_norm_rope(s)
            return q.to(s["q"].dtype), k.to(s["q"].dtype)
        if kind == "fused":
            q, k = _plain_norm_rope(s)
            return q.to(s["q"].dtype), _plain_store(s, "k", k), _plain_store(s, "v", s["v"])
        if kind == "store":
            return _plain_store(s, "k", s["k"]), _plain_store(s, "v", s["v"])
        return _plain_load(s)
    from sglang_b200.layers import lora, rotary_embedding
    from sglang_b200.layers.quantization import kv_cache
    if kind == "lora":
        return lora.apply_lora(s["base"], s["x"], s["lora_a"], s["lora_b"], s["batch"], output_sizes=s["sizes"], out=s["out"])
    if kind == "norm_rope":
        return rotary_embedding.qk_norm_rope(s["q"], s["k"], s["positions"], s["cos_sin"], s["q_weight"], s["k_weight"],
                                             norm_eps=EPS, is_neox=s["neox"])
    if kind == "load":
        return kv_cache.load_kv_fp8(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["page_table"], s["indptr"],
                                    s["tokens"], out_dtype=s["dtype"])
    held = (s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])
    if kind == "store":
        kv_cache.store_kv_fp8(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["slots"])
        return held
    q = kv_cache.qk_norm_rope_store_kv_fp8(s["q"], s["k"], s["v"], s["positions"], s["cos_sin"], s["k_cache"], s["v_cache"],
                                           s["k_scale"], s["v_scale"], s["slots"], s["q_weight"], s["k_weight"],
                                           norm_eps=EPS, is_neox=s["neox"])
    return (q,) + held


# ------------------------------------------------------------------------------------------------------- what it is
def work(case):
    T, kind = case["T"], case["kind"]
    if kind == "lora":
        sizes = [int(n) for n in case["sizes"].split(",")]
        K, R, N, S = case["K"], case["R"], sum(sizes), len(sizes)
        used = min(case["L"], case["segments"])
        rank = sum(max(1, R >> (a % 3)) for a in range(used)) / used      # of an adapter, on average
        share = 1 - case["bare"]
        read = T * K * share + T * N + used * rank * (S * K + N)
        return {"bytes": 2 * (read + T * N), "flops": 2 * T * share * rank * (S * K + N)}
    row = case["Hkv"] * case["D"]
    held = T * 2 * (row + 4 * case["Hkv"])            # codes and scales of T tokens, keys and values
    if kind == "load":
        return {"bytes": held + T * 4 * row, "flops": T * 2 * row}
    if kind == "store":
        return {"bytes": held + T * 4 * row + 8 * T, "flops": T * 6 * row}
    turned = T * (case["Hq"] + case["Hkv"]) * case["D"]
    table = T * (4 * case["rot"] + 8)
    if kind == "norm_rope":
        return {"bytes": 4 * turned + table, "flops": 7 * turned}
    return {"bytes": 2 * turned + 2 * T * row + 2 * T * case["Hq"] * case["D"] + held + table + 8 * T,
            "flops": 7 * turned + T * 6 * row}


def _exact_rows(x, weight, turn, neox):
    """The first elements of each head as complex numbers, multiplied with the token's row of `turn`."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    half = turn.shape[1]
    y = x.clone()
    first = torch.arange(half, device=x.device) * (1 if neox else 2)
    second = first + (half if neox else 1)
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_codes(x):
    """(the e4m3 number nearest to each x / scale, ties to even; scale), a scale for each row's largest magnitude."""
    scale = torch.clamp(x.abs().max(-1).values, min=1e-10) / 448
    v = x / scale[..., None]
    step = torch.exp2(torch.clamp(torch.frexp(v.abs()).exponent - 1, min=-6).double() - 3)
    return torch.clamp(torch.round(v / step) * step, -448, 448), scale


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "lora":
        out, R, ends = s["base"].double(), case["R"], [0]
        for n in s["sizes"]:
            ends.append(ends[-1] + n)
        for a, (rank, scaling) in enumerate(zip(s["ranks"].tolist(), s["scalings"].tolist())):
            rows = (s["ids"] == a).nonzero().flatten()
            for i in range(len(s["sizes"])):
                A, B = s["lora_a"][a, i * R:i * R + rank].double(), s["lora_b"][a, ends[i]:ends[i + 1], :rank].double()
                out[rows, ends[i]:ends[i + 1]] += scaling * (s["x"][rows].double() @ A.T) @ B.T
        return out
    if kind == "load":
        page, indptr = case["page"], s["indptr"].tolist()
        found = []
        for n in ("k", "v"):
            rows = []
            for b in range(len(indptr) - 1):
                count = indptr[b + 1] - indptr[b]
                pages = s["page_table"][b, :(count + page - 1) // page].long()
                codes = s[n + "_cache"].view(torch.uint8)[pages].view(FP8)
                rows.append((codes.double() * s[n + "_scale"][pages].double()[..., None]).flatten(0, 1)[:count])
            found.append(torch.cat(rows))
        return tuple(found)
    kept = {}
    if kind != "store":
        turn = torch.complex(*s["cos_sin"].double()[s["positions"]].chunk(2, dim=1))
        q = _exact_rows(s["q"], s["q_weight"], turn, case["neox"])
        k = _exact_rows(s["k"], s["k_weight"], turn, case["neox"])
        if kind == "norm_rope":
            return q, k
        kept["k"] = k
    else:
        kept["k"] = s["k"].double()
    kept["v"] = s["v"].double()
    held = []
    for n in ("k", "v"):
        cache, scales = s[n + "_cache"].double(), s[n + "_scale"].double()
        new, scale = _exact_codes(kept[n])
        cache.flatten(0, 1)[s["slots"]] = new
        scales.flatten(0, 1)[s["slots"]] = scale
        held.append((cache, scales))
    return ((q,) if kind == "fused" else ()) + tuple(held)
