"""What is measured of the language-model operators: four operators of one attention layer's serving step, through the entry
points that a program calls, and the same in elementary torch operations.

  int8    a dense layer in 8-bit integers with a scale for each token and each output channel.  Activations of 16 or 32 bits
          are brought to 8 bits token by token first (pb_int8_quantize_launch), then multiplied (pb_int8_dense_launch).
  rope    norms of queries and keys for each head and the rotation by position (pb_qk_rope_launch)
  append  keys and values into a paged cache, keys normed and rotated on the way, the step's queries beside them
          (pb_kv_append_launch)
  attn    one new token of every sequence of a batch that shares a long prefix, over the paged cache (pb_prefix_attn_launch)

`listed()` are the cases themselves, `draw()` gives more of the same ranges.
"""
import ctypes as C
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "s8": torch.int8}
CODES = {"f32": 0, "bf16": 1, "f16": 2, "s8": 3}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "s8": 1}
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------

def _int8(t, k, n, x="bf16", y="bf16", bias=False, act=0):
    return {"op": "int8", "t": t, "k": k, "n": n, "x": x, "y": y, "bias": bias, "act": act}


def _rope(t, hq, hkv, d, rot, dtype="bf16", interleaved=False, norm=True):
    return {"op": "rope", "t": t, "hq": hq, "hkv": hkv, "d": d, "rot": rot, "dtype": dtype, "interleaved": interleaved, "norm": norm}


def _append(t, hq, hkv, d, rot, page, pages, dtype="bf16", interleaved=False, norm=True, heads_first=False, padded=0):
    return {"op": "append", "t": t, "hq": hq, "hkv": hkv, "d": d, "rot": rot, "page": page, "pages": pages, "dtype": dtype,
            "interleaved": interleaved, "norm": norm, "heads_first": heads_first, "padded": padded}


def _attn(b, hkv, g, d, prefix, most, page, dtype="bf16", heads_first=False):
    return {"op": "attn", "b": b, "hkv": hkv, "g": g, "d": d, "prefix": prefix, "most": most, "page": page, "dtype": dtype,
            "heads_first": heads_first}


def listed():
    return [
        # One user's next token through a square projection: the weights are read for a single row, latency counts.
        {"name": "int8_1_token", **_int8(1, 4096, 4096)},
        # A decode batch through a widening layer, with its bias.
        {"name": "int8_24_tokens", **_int8(24, 4096, 14336, bias=True)},
        # A prompt's chunk of any length through a layer of odd width, activations already in 8 bits, fp32 results, relu.
        {"name": "int8_ragged", **_int8(777, 2000, 5001, x="s8", y="f32", bias=True, act=1)},
        # A full prefill batch: arithmetic alone counts.
        {"name": "int8_8192_tokens", **_int8(8192, 8192, 8192, x="f16", y="f16")},
        # A decode batch's queries and keys, four query heads a key head.
        {"name": "rope_48_tokens", **_rope(48, 32, 8, 128, 128)},
        # A prefill batch, larger than the L2 cache.
        {"name": "rope_16384_tokens", **_rope(16384, 32, 8, 128, 128)},
        # One user's next token into the cache: the smallest call there is.
        {"name": "append_1_token", **_append(1, 32, 8, 128, 128, 16, 256)},
        # A padded prefill batch: 200 rows belong to no sequence, part of each head is rotated, pairs lie side by side, no norm.
        {"name": "append_padded", **_append(9001, 24, 6, 96, 64, 64, 256, dtype="f16", interleaved=True, norm=False, heads_first=True, padded=200)},
        # Four short answers to one prompt on a small model: latency counts.
        {"name": "attn_4_short", **_attn(4, 2, 4, 64, 300, 20, 16)},
        # A decode batch behind a system prompt.
        {"name": "attn_32", **_attn(32, 8, 4, 128, 8192, 512, 32)},
        # Sixteen samples from one very long document, whose length ends inside a page: the cache's bytes count.
        {"name": "attn_long_prefix", **_attn(16, 8, 8, 128, 130001, 700, 64)},
        # A large batch of grouped heads: arithmetic over the prefix, bytes behind it.
        {"name": "attn_256", **_attn(256, 8, 8, 128, 16384, 1024, 64, dtype="f16")},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("int8", "rope", "append", "attn"))
    if op == "int8":
        while True:
            t, k, n = _log(rng, 1, 8192), _log(rng, 64, 16384), _log(rng, 64, 16384)
            if t * k * n <= 8192 ** 3 // 2:
                break
        x = rng.choice(("bf16", "f16", "f32", "s8"))
        return _int8(t, k, n, x, rng.choice(("bf16", "f16", "f32")), rng.random() < 0.5, rng.choice((0, 0, 1)))
    d = rng.choice((64, 80, 96, 128))
    hkv, g = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 5, 8))
    dtype = rng.choice(("bf16", "f16"))
    if op == "attn":
        b, prefix, most = _log(rng, 1, 256), _log(rng, 1, 65536), _log(rng, 1, 2048)
        while b * g * hkv * (prefix + most) > 256 * 8 * 8 * 8192 or b * most * hkv > 256 * 512 * 8:
            b, prefix, most = _log(rng, 1, 256), _log(rng, 1, 65536), _log(rng, 1, 2048)
        return _attn(b, hkv, g, d, prefix, most, rng.choice((16, 32, 64, 128)), dtype, rng.random() < 0.5)
    rot = rng.choice((d, d, d // 2))
    if rng.random() < 0.2:
        dtype = "f32"
    if op == "rope":
        return _rope(_log(rng, 1, 16384), g * hkv, hkv, d, rot, dtype, rng.random() < 0.3, rng.random() < 0.7)
    t, page = _log(rng, 1, 8192), rng.choice((16, 32, 64, 128))
    return _append(t, rng.choice((0, g * hkv)), hkv, d, rot, page, -(-t // page) + rng.randint(8, 64), dtype, rng.random() < 0.3,
                   rng.random() < 0.7, rng.random() < 0.5, rng.choice((0, t // 16)))


# ---------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _rotation_table(positions, rot):
    """cosines, then sines, of every position up to the last: angles in 64 bits, each function rounded once"""
    at = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None]
    angle = at * 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


def _own_lengths(case):
    """tokens behind the prefix, from none to the most"""
    b = case["b"]
    return [case["most"] * (i + 1) // b if b < 3 else case["most"] * i // (b - 1) for i in range(b)]


def _cache(gen, case, pages):
    """keys and values as [pages][page][heads][d], or with the heads in front of the tokens of a page"""
    inner = (case["hkv"], case["page"]) if case["heads_first"] else (case["page"], case["hkv"])
    return [_randn(gen, pages, *inner, case["d"]).to(TYPES[case["dtype"]]) for _ in range(2)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case, "keep": {}}
    if case["op"] == "int8":
        t, k, n = case["t"], case["k"], case["n"]
        row = -(-k // 16) * 16                       # rows of 8-bit operands start on 16 bytes
        x = _randn(gen, t, k)
        if case["x"] == "s8":
            st["x"] = torch.zeros(t, row, dtype=torch.int8, device="cuda")
            st["x"][:, :k] = (x * 42.0).round().clamp(-127, 127).to(torch.int8)
            st["x_scale"] = torch.rand(t, generator=gen, device="cuda") * 0.03 + 0.01
        else:
            x *= torch.exp(0.5 * _randn(gen, t, 1))  # tokens of different size
            st["x"] = x.to(TYPES[case["x"]])
        st["w"] = torch.zeros(n, row, dtype=torch.int8, device="cuda")
        st["w"][:, :k] = torch.randint(-127, 128, (n, k), generator=gen, device="cuda", dtype=torch.int8)
        st["w_scale"] = (torch.rand(n, generator=gen, device="cuda") + 0.5) / (73.0 * math.sqrt(k))
        st["bias"] = _randn(gen, n) * 0.1 if case["bias"] else None
        return st
    d = case["d"]
    if case["op"] == "attn":
        b, page, g, hkv = case["b"], case["page"], case["g"], case["hkv"]
        lengths = _own_lengths(case)
        ahead, each = -(-case["prefix"] // page), -(-case["most"] // page)
        pages = ahead + b * each + 3
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        st["k_cache"], st["v_cache"] = _cache(gen, case, pages)
        st["prefix_pages"] = order[:ahead].contiguous()
        st["block_table"] = order[ahead:ahead + b * each].view(b, each).contiguous()
        mix = torch.randperm(b, generator=gen, device="cuda")
        st["own_lens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")[mix].contiguous()
        st["q"] = (1.5 * _randn(gen, b, hkv * g, d)).to(TYPES[case["dtype"]])
        return st
    t, hq, hkv, ty = case["t"], case["hq"], case["hkv"], TYPES[case["dtype"]]
    # queries, keys and values as a projection leaves them: one row for each token
    heads = hq + hkv * (2 if case["op"] == "append" else 1)
    rows = _randn(gen, t, heads, d).to(ty)
    st["q"], st["k"] = rows[:, :hq], rows[:, hq:hq + hkv]
    st["max_position"] = 32768
    st["table"] = _rotation_table(st["max_position"], case["rot"])
    st["positions"] = torch.randint(0, st["max_position"], (t,), generator=gen, device="cuda", dtype=torch.int32)
    st["q_weight"] = 1.0 + 0.1 * _randn(gen, d) if case["norm"] else None
    st["k_weight"] = 1.0 + 0.1 * _randn(gen, d) if case["norm"] else None
    if case["op"] == "append":
        st["v"] = rows[:, hq + hkv:]
        st["k_cache"], st["v_cache"] = _cache(gen, case, case["pages"])
        slots = torch.randperm(case["pages"] * case["page"], generator=gen, device="cuda")[:t]
        if case["padded"]:
            slots[t - case["padded"]:] = -1
        st["slots"] = slots.contiguous()
    return st


# ---------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------

def _plain_int8(case, st):
    k = case["k"]
    if case["x"] == "s8":
        x, scale = st["x"][:, :k].float(), st["x_scale"]
    else:
        x = st["x"].float()
        most = x.abs().amax(1)
        x = (x * (127.0 / most)[:, None]).round()
        scale = most / 127.0
    y = (x @ st["w"][:, :k].float().t()) * scale[:, None] * st["w_scale"]
    if st["bias"] is not None:
        y = y + st["bias"]
    if case["act"] == 1:
        y = y.relu()
    return y.to(TYPES[case["y"]])


def _plain_heads(case, x, weight, table, positions):
    """norm and rotation of [tokens][heads][d]"""
    ty, rot = x.dtype, case["rot"]
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    both = table[positions.long()][:, None]
    c, s = both[..., :rot // 2], both[..., rot // 2:]
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, x[..., rot:]], -1).to(ty)


def _plain_rope(case, st):
    return (_plain_heads(case, st["q"], st["q_weight"], st["table"], st["positions"]),
            _plain_heads(case, st["k"], st["k_weight"], st["table"], st["positions"]))


def _plain_append(case, st):
    k = _plain_heads(case, st["k"], st["k_weight"], st["table"], st["positions"])
    v, slots, page = st["v"], st["slots"], case["page"]
    if case["padded"]:
        real = slots >= 0
        k, v, slots = k[real], v[real], slots[real]
    kc, vc = st["k_cache"], st["v_cache"]
    if case["heads_first"]:
        kc[slots // page, :, slots % page] = k
        vc[slots // page, :, slots % page] = v
    else:
        kc.view(-1, *kc.shape[2:])[slots] = k
        vc.view(-1, *vc.shape[2:])[slots] = v
    q = _plain_heads(case, st["q"], st["q_weight"], st["table"], st["positions"]) if case["hq"] else None
    return kc, vc, q


def _tokens(case, cache, table):
    """the tokens of the pages in `table`, as [..., pages * page][heads][d] in 32 bits"""
    got = cache[table.long()].float()
    if case["heads_first"]:
        got = got.transpose(-2, -3)
    return got.flatten(-4, -3)


def _plain_attn(case, st):
    b, hkv, g, d, n = case["b"], case["hkv"], case["g"], case["d"], case["prefix"]
    q = st["q"].float().view(b, hkv, g, d) * d ** -0.5
    k = _tokens(case, st["k_cache"], st["prefix_pages"])[:n]
    s_prefix = torch.matmul(q.permute(1, 0, 2, 3).reshape(hkv, b * g, d), k.permute(1, 2, 0)).view(hkv, b, g, n).transpose(0, 1)
    k = _tokens(case, st["k_cache"], st["block_table"])
    s_own = torch.matmul(q, k.permute(0, 2, 3, 1))
    seen = torch.arange(k.shape[1], device="cuda") < st["own_lens"][:, None]
    s_own = s_own.masked_fill(~seen[:, None, None], -math.inf)
    del k
    top = torch.maximum(s_prefix.amax(-1), s_own.amax(-1))[..., None]
    p_prefix, p_own = torch.exp(s_prefix - top), torch.exp(s_own - top)
    total = p_prefix.sum(-1) + p_own.sum(-1)
    v = _tokens(case, st["v_cache"], st["prefix_pages"])[:n]
    out = torch.matmul(p_prefix.transpose(0, 1).reshape(hkv, b * g, n), v.transpose(0, 1)).view(hkv, b, g, d).transpose(0, 1)
    v = _tokens(case, st["v_cache"], st["block_table"]).masked_fill(~seen[:, :, None, None], 0.0)
    out = out + torch.matmul(p_own, v.transpose(1, 2))
    return (out / total[..., None]).reshape(b, hkv * g, d).to(TYPES[case["dtype"]])


# ---------------------------------------------------------------------------------------------------
# The framework's calls.  A program fills an operator's parameters once for the buffers it keeps, and launches.
# ---------------------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_int8(case, st, keep):
    from paella_b200 import capi
    L, t, k, n = capi.load(), case["t"], case["k"], case["n"]
    x, scale, launches = st["x"], st.get("x_scale"), []
    if case["x"] != "s8":
        x, scale = torch.empty(t, st["w"].shape[1], dtype=torch.int8, device="cuda"), torch.empty(t, device="cuda")
        p = capi.Int8QuantizeParams(tokens=t, channels=k, x_dtype=CODES[case["x"]], x_stride=st["x"].stride(0), q_stride=x.stride(0),
                                    x=_ptr(st["x"]), q=_ptr(x), scale=_ptr(scale))
        launches.append((L.pb_int8_quantize_launch, p))
    y = torch.empty(t, n, dtype=TYPES[case["y"]], device="cuda")
    p = capi.Int8DenseParams(tokens=t, in_channels=k, out_channels=n, y_dtype=CODES[case["y"]], act=case["act"], x_stride=x.stride(0),
                             w_stride=st["w"].stride(0), y_stride=n, x=_ptr(x), x_scale=_ptr(scale), w=_ptr(st["w"]),
                             w_scale=_ptr(st["w_scale"]), bias=_ptr(st["bias"]), y=_ptr(y))
    launches.append((L.pb_int8_dense_launch, p))
    keep.update(launches=launches, out=y, buffers=(x, scale))


def _own_rope(case, st, keep):
    from paella_b200 import capi
    L, q, k = capi.load(), st["q"], st["k"]
    q_out, k_out = torch.empty(q.shape, dtype=q.dtype, device="cuda"), torch.empty(k.shape, dtype=k.dtype, device="cuda")
    p = capi.QkRopeParams(dtype=CODES[case["dtype"]], tokens=case["t"], q_heads=case["hq"], kv_heads=case["hkv"], head_dim=case["d"],
                          rot_dim=case["rot"], interleaved=int(case["interleaved"]), max_position=st["max_position"], eps=EPS,
                          q_stride=q.stride(0), q_head_stride=q.stride(1), k_stride=k.stride(0), k_head_stride=k.stride(1),
                          q_out_stride=q_out.stride(0), q_out_head_stride=q_out.stride(1), k_out_stride=k_out.stride(0),
                          k_out_head_stride=k_out.stride(1), q=_ptr(q), k=_ptr(k), q_out=_ptr(q_out), k_out=_ptr(k_out),
                          q_weight=_ptr(st["q_weight"]), k_weight=_ptr(st["k_weight"]), cos_sin=_ptr(st["table"]),
                          positions=_ptr(st["positions"]))
    keep.update(launches=[(L.pb_qk_rope_launch, p)], out=(q_out, k_out))


def _own_append(case, st, keep):
    from paella_b200 import capi
    L, q, k, v, kc, vc = capi.load(), st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"]
    q_out = torch.empty(q.shape, dtype=q.dtype, device="cuda") if case["hq"] else None
    token, head = (kc.stride(2), kc.stride(1)) if case["heads_first"] else (kc.stride(1), kc.stride(2))
    p = capi.KvAppendParams(dtype=CODES[case["dtype"]], tokens=case["t"], q_heads=case["hq"], kv_heads=case["hkv"], head_dim=case["d"],
                            rot_dim=case["rot"], interleaved=int(case["interleaved"]), max_position=st["max_position"], eps=EPS,
                            page_size=case["page"], n_pages=kc.shape[0], k_stride=k.stride(0), k_head_stride=k.stride(1),
                            v_stride=v.stride(0), v_head_stride=v.stride(1), page_stride=kc.stride(0), token_stride=token,
                            head_stride=head, k=_ptr(k), v=_ptr(v), k_weight=_ptr(st["k_weight"]), cos_sin=_ptr(st["table"]),
                            positions=_ptr(st["positions"]), slots=_ptr(st["slots"]), k_cache=_ptr(kc), v_cache=_ptr(vc))
    if case["hq"]:
        p.q_stride, p.q_head_stride, p.q_out_stride, p.q_out_head_stride = q.stride(0), q.stride(1), q_out.stride(0), q_out.stride(1)
        p.q, p.q_out, p.q_weight = _ptr(q), _ptr(q_out), _ptr(st["q_weight"])
    keep.update(launches=[(L.pb_kv_append_launch, p)], out=(kc, vc, q_out))


def _own_attn(case, st, keep):
    from paella_b200 import capi
    L, q, kc, table = capi.load(), st["q"], st["k_cache"], st["block_table"]
    out = torch.empty_like(q)
    token, head = (kc.stride(2), kc.stride(1)) if case["heads_first"] else (kc.stride(1), kc.stride(2))
    p = capi.PrefixAttnParams(dtype=CODES[case["dtype"]], batch=case["b"], q_heads=q.shape[1], kv_heads=case["hkv"],
                              head_dim=case["d"], page_size=case["page"], max_blocks=table.shape[1], prefix_len=case["prefix"],
                              max_own_len=case["most"], scale=case["d"] ** -0.5, n_pages=kc.shape[0], q_stride=q.stride(0),
                              q_head_stride=q.stride(1), out_stride=out.stride(0), out_head_stride=out.stride(1),
                              page_stride=kc.stride(0), token_stride=token, head_stride=head, table_stride=table.stride(0),
                              q=_ptr(q), out=_ptr(out), k_cache=_ptr(kc), v_cache=_ptr(st["v_cache"]),
                              prefix_pages=_ptr(st["prefix_pages"]), block_table=_ptr(table), own_lens=_ptr(st["own_lens"]))
    info = capi.LaunchInfo()
    capi.check(L.pb_prefix_attn_info(C.byref(p), C.byref(info)), "pb_prefix_attn_info")
    scratch = torch.empty(max(16, info.scratch_bytes), dtype=torch.uint8, device="cuda")
    p.scratch, p.scratch_bytes = _ptr(scratch), info.scratch_bytes
    keep.update(launches=[(L.pb_prefix_attn_launch, p)], out=out, buffers=scratch)


def run(st):
    case = st["case"]
    if own:
        keep = st["keep"]
        if not keep:
            {"int8": _own_int8, "rope": _own_rope, "append": _own_append, "attn": _own_attn}[case["op"]](case, st, keep)
        stream = torch.cuda.current_stream().cuda_stream
        for launch, p in keep["launches"]:
            rc = launch(C.byref(p), stream, 0, None)
            if rc != 0:
                from paella_b200 import capi
                capi.check(rc, launch.__name__)
        return keep["out"]
    return {"int8": _plain_int8, "rope": _plain_rope, "append": _plain_append, "attn": _plain_attn}[case["op"]](case, st)


# ---------------------------------------------------------------------------------------------------
# What a pass cannot do without, and what it comes to in 64 bits
# ---------------------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "int8":
        t, k, n = case["t"], case["k"], case["n"]
        return {"bytes": t * k * BYTES[case["x"]] + n * k + 4 * n * (2 if case["bias"] else 1) + (4 * t if case["x"] == "s8" else 0) +
                t * n * BYTES[case["y"]], "flops": 2 * t * k * n}
    es, d, hkv = BYTES[case["dtype"]], case["d"], case["hkv"]
    if case["op"] == "attn":
        tokens, rows = sum(_own_lengths(case)), case["b"] * case["g"]
        return {"bytes": es * d * (2 * hkv * (case["prefix"] + tokens) + 2 * rows * hkv) + 4 * (case["b"] + -(-case["prefix"] // case["page"])),
                "flops": 4 * d * hkv * case["g"] * (case["b"] * case["prefix"] + tokens)}
    t = case["t"] - case.get("padded", 0)
    # a row of the rotation table for every token, which far positions spread over the whole of it
    heads = case["hq"] + hkv * (2 if case["op"] == "append" else 1)
    return {"bytes": 2 * t * heads * d * es + t * (4 * case["rot"] + 4 + (8 if case["op"] == "append" else 0)),
            "flops": t * (case["hq"] + hkv) * (3 * case["rot"] + (4 * d if case["norm"] else 0))}


def _exact_heads(case, x, weight, st):
    """each head on its own: complex numbers turned by the table's angles"""
    x, rot = x.double(), case["rot"]
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / case["d"] + EPS).sqrt() * weight.double()
    row = st["table"].double()[st["positions"].long()]
    turn = torch.complex(row[:, :rot // 2], row[:, rot // 2:]).unsqueeze(1)
    even, odd = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    z = torch.complex(x[..., even], x[..., odd]) * turn
    out = x.clone()
    out[..., even], out[..., odd] = z.real, z.imag
    return out


def _exact_attn(case, st):
    b, hkv, g, d, page = case["b"], case["hkv"], case["g"], case["d"], case["page"]

    def token(cache, pages, n):
        at = torch.arange(n, device="cuda")
        page_of, row = pages.long()[at // page], at % page
        return (cache[page_of, :, row] if case["heads_first"] else cache[page_of, row]).double()

    q = st["q"].double()
    k0, v0 = (token(st[c], st["prefix_pages"], case["prefix"]) for c in ("k_cache", "v_cache"))
    out = torch.empty(b, hkv * g, d, dtype=torch.float64, device="cuda")
    lengths = st["own_lens"].tolist()
    own_kv = [[token(st[c], st["block_table"][i], lengths[i]) for c in ("k_cache", "v_cache")] for i in range(b)]
    for h in range(hkv):
        heads = slice(h * g, (h + 1) * g)
        first = (q[:, heads].reshape(b * g, d) @ k0[:, h].t() / math.sqrt(d)).view(b, g, -1)
        seconds = [q[i, heads] @ own_kv[i][0][:, h].t() / math.sqrt(d) for i in range(b)]
        top = torch.stack([torch.cat([first[i], seconds[i]], 1).amax(1) for i in range(b)])
        first = torch.exp(first - top[..., None])
        total, acc = first.sum(-1), (first.view(b * g, -1) @ v0[:, h]).view(b, g, d)
        for i in range(b):
            e = torch.exp(seconds[i] - top[i][:, None])
            total[i] += e.sum(1)
            acc[i] += e @ own_kv[i][1][:, h]
        out[:, heads] = acc / total[..., None]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "int8":
        k = case["k"]
        if case["x"] == "s8":
            x, scale = st["x"][:, :k], st["x_scale"].double()
        else:
            # the 8-bit integers are by definition those that the 32-bit product with 127 / max rounds to
            most = st["x"].float().abs().amax(1)
            x, scale = torch.round(st["x"].float() * (127.0 / most)[:, None]), most.double() / 127
        y = torch.einsum("tk,nk->tn", x.double(), st["w"][:, :k].double()) * torch.outer(scale, st["w_scale"].double())
        if st["bias"] is not None:
            y += st["bias"].double()
        return y.clamp_min(0) if case["act"] == 1 else y
    if case["op"] == "attn":
        return _exact_attn(case, st)
    q = _exact_heads(case, st["q"], st["q_weight"], st) if case["hq"] else None
    k = _exact_heads(case, st["k"], st["k_weight"], st)
    if case["op"] == "rope":
        return q, k
    kc, vc, page = st["k_cache"].double(), st["v_cache"].double(), case["page"]
    real = torch.nonzero(st["slots"] >= 0).flatten()
    at = st["slots"][real]
    where = (at // page, slice(None), at % page) if case["heads_first"] else (at // page, at % page)
    kc[where], vc[where] = k[real], st["v"][real].double()
    return kc, vc, q
