"""What is measured of the operators that take a prompt through a language model and say what it made of it, beside those of
`operators.py`: through the entry points that a program calls, and the same in elementary torch operations.

  chunk     attention of each sequence's new tokens, one or many, over a paged cache that holds them already (pb_chunk_attn_launch)
  norm      a block's output normed, gated, scaled and added to the residual, and the norm in front of the next block
            (pb_residual_norm_launch)
  logprobs  log probability and rank of a given token for each row of logits, the row's entropy and its likeliest tokens
            (pb_logprobs_launch)

`listed()` are the cases themselves, `draw()` gives more of the same ranges.
"""
import ctypes as C
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"f32": 0, "bf16": 1, "f16": 2}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------

def _chunk(b, new, ctx, hkv, g, d, page, dtype="bf16", mixed=False, window=0, heads_first=False, padded=0):
    return {"op": "chunk", "b": b, "new": new, "ctx": ctx, "hkv": hkv, "g": g, "d": d, "page": page, "dtype": dtype, "mixed": mixed,
            "window": window, "heads_first": heads_first, "padded": padded}


def _norm(t, c, dtype="bf16", stream="same", post=False, gate="none"):
    return {"op": "norm", "t": t, "c": c, "dtype": dtype, "stream": stream, "post": post, "gate": gate}


def _logprobs(t, v, top, dtype="bf16", scale=1.0, kept=1.0):
    return {"op": "logprobs", "t": t, "v": v, "top": top, "dtype": dtype, "scale": scale, "kept": kept}


def listed():
    return [
        # A small model's decode batch, one token each, without a prefix to share: latency counts.
        {"name": "chunk_8_decode", **_chunk(8, 1, 2000, 2, 4, 64, 16)},
        # Four guessed tokens of every sequence of a decode batch, to be verified: the cache's bytes count.
        {"name": "chunk_24_verify", **_chunk(24, 4, 4096, 8, 4, 128, 32)},
        # One prompt from its first token on.
        {"name": "chunk_prompt", **_chunk(1, 8192, 0, 8, 4, 128, 64)},
        # A serving step that takes chunks of some prompts along with the next token of many sequences, under a sliding window,
        # with rows behind the last sequence.
        {"name": "chunk_mixed", **_chunk(64, 1024, 3000, 6, 5, 96, 16, dtype="f16", mixed=True, window=1024, heads_first=True, padded=40)},
        # The next chunk of a long document: arithmetic over the cache.
        {"name": "chunk_long", **_chunk(1, 2048, 65000, 8, 4, 128, 64)},
        # One user's next token between two blocks: the smallest call there is.
        {"name": "norm_1_token", **_norm(1, 4096)},
        # A prompt's chunk of any length through a block of odd width, with a gate for each token and the residual kept in 32 bits.
        {"name": "norm_ragged", **_norm(777, 5001, "f16", "f32", True, "token")},
        # A prefill batch, larger than the L2 cache, norms on both sides of the block and one gate for all tokens.
        {"name": "norm_16384_tokens", **_norm(16384, 4096, "bf16", "same", True, "channel")},
        # A decode batch that asks for the twenty likeliest tokens: few long rows.
        {"name": "logprobs_4_rows", **_logprobs(4, 131072, 20, "f32", 1.25)},
        # A prompt's chunk under a mask that leaves a tenth of an odd vocabulary.
        {"name": "logprobs_masked", **_logprobs(333, 50001, 5, "bf16", 0.7, 0.1)},
        # A prompt that is scored: nothing but its own tokens.
        {"name": "logprobs_scored", **_logprobs(4096, 32000, 0, "f16")},
        # The same over a large vocabulary, with alternatives.
        {"name": "logprobs_2048_rows", **_logprobs(2048, 131072, 5)},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("chunk", "norm", "logprobs"))
    if op == "chunk":
        most = work(listed()[4])
        while True:
            case = _chunk(_log(rng, 1, 256), rng.choice((1, _log(rng, 1, 8192))), _log(rng, 1, 65536) - 1, rng.choice((1, 2, 4, 8)),
                          rng.choice((1, 2, 3, 4, 5, 8)), rng.choice((64, 80, 96, 128)), rng.choice((16, 32, 64, 128)),
                          rng.choice(("bf16", "f16")), rng.random() < 0.4, rng.choice((0, 0, _log(rng, 16, 8192))), rng.random() < 0.5,
                          rng.choice((0, _log(rng, 1, 100))))
            cost = work(case)
            # a window leaves most of a cache unread, which is made all the same
            kept = sum(n + ctx for n, ctx in _lengths(case)) * case["hkv"] * case["d"]
            if cost["flops"] <= most["flops"] / 2 and cost["bytes"] <= 2 << 30 and kept <= 1 << 29:
                return case
    if op == "norm":
        while True:
            t, c = _log(rng, 1, 16384), _log(rng, 64, 16384)
            if t * c <= 16384 * 4096 // 2:
                break
        dtype = rng.choice(("bf16", "f16", "f32"))
        return _norm(t, c, dtype, rng.choice(("same", "f32")), rng.random() < 0.5, rng.choice(("none", "token", "channel")))
    while True:
        t, v = _log(rng, 1, 8192), _log(rng, 1000, 262144)
        if t * v <= 2048 * 131072 // 2:
            break
    return _logprobs(t, v, rng.choice((0, 1, 5, 20, 32)), rng.choice(("bf16", "f16", "f32")), rng.choice((1.0, 1.25, 0.7)),
                     rng.choice((1.0, 1.0, 0.1)))


# ---------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _lengths(case):
    """(new tokens, tokens in front of them) of every sequence"""
    b = case["b"]
    new = [1 if case["mixed"] and i % 8 else -(-case["new"] * (b - i) // b) for i in range(b)]
    return [(n, case["ctx"] if b == 1 else case["ctx"] * i // (b - 1)) for i, n in enumerate(new)]


def _prepare_chunk(case, gen, st):
    b, page, hkv, d, ty = case["b"], case["page"], case["hkv"], case["d"], TYPES[case["dtype"]]
    mix = torch.randperm(b, generator=gen, device="cuda").tolist()
    lengths = [_lengths(case)[i] for i in mix]
    st["max_len"] = max(n + ctx for n, ctx in lengths)
    each = -(-st["max_len"] // page)
    used = [-(-(n + ctx) // page) for n, ctx in lengths]
    pages = sum(used) + 3
    inner = (hkv, page) if case["heads_first"] else (page, hkv)
    st["k_cache"], st["v_cache"] = (_randn(gen, pages, *inner, d).to(ty) for _ in range(2))
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table, at = torch.zeros(b, each, dtype=torch.int32, device="cuda"), 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    st["block_table"] = table
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    st["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    st["lens"] = torch.tensor([n + ctx for n, ctx in lengths], dtype=torch.int32, device="cuda")
    st["host"] = [(starts[i], n, n + ctx) for i, (n, ctx) in enumerate(lengths)]
    tokens = starts[-1] + case["padded"]
    st["q"] = (1.5 * _randn(gen, tokens, hkv * case["g"], d)).to(ty)
    st["out"] = _randn(gen, tokens, hkv * case["g"], d).to(ty)       # rows of no sequence stay as they are


def _prepare_norm(case, gen, st):
    t, c, ty = case["t"], case["c"], TYPES[case["dtype"]]
    stream = torch.float32 if case["stream"] == "f32" else ty
    st["x"] = (_randn(gen, t, c) * torch.exp(0.5 * _randn(gen, t, 1))).to(ty)
    st["residual"] = (4.0 * _randn(gen, t, c)).to(stream)
    st["post_weight"] = 1.0 + 0.1 * _randn(gen, c) if case["post"] else None
    st["weight"] = 1.0 + 0.1 * _randn(gen, c)
    rows = {"none": 0, "channel": 1, "token": t}[case["gate"]]
    st["gate"] = torch.sigmoid(_randn(gen, rows, c)).to(ty) if rows else None
    st["scale"] = 0.5


def _prepare_logprobs(case, gen, st):
    t, v, ty = case["t"], case["v"], TYPES[case["dtype"]]
    logits = torch.empty(t, v, dtype=ty, device="cuda")
    targets = torch.randint(0, v, (t,), generator=gen, device="cuda")
    for a in range(0, t, 512):
        x = 2.5 * _randn(gen, min(512, t - a), v)
        # what a model is sure of: a few tokens far above the others
        sure = torch.randint(0, v, (x.shape[0], 4), generator=gen, device="cuda")
        x.scatter_add_(1, sure, 4.0 * _randn(gen, x.shape[0], 4).abs() + 6.0)
        if case["kept"] < 1.0:
            x.masked_fill_(torch.rand(x.shape, generator=gen, device="cuda") >= case["kept"], -math.inf)
        right = torch.rand(x.shape[0], generator=gen, device="cuda") < 0.5
        targets[a:a + 512] = torch.where(right, x.argmax(1), targets[a:a + 512])
        rows = torch.arange(x.shape[0], device="cuda")
        mine = x[rows, targets[a:a + 512]]
        x[rows, targets[a:a + 512]] = torch.where(mine == -math.inf, 0.5, mine)
        logits[a:a + 512] = x.to(ty)
    st["logits"], st["targets"] = logits, targets.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case, "keep": {}}
    {"chunk": _prepare_chunk, "norm": _prepare_norm, "logprobs": _prepare_logprobs}[case["op"]](case, gen, st)
    return st


# ---------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------

def _plain_chunk(case, st):
    hkv, g, d, page = case["hkv"], case["g"], case["d"], case["page"]
    out = st["out"].clone()
    for i, (start, n, length) in enumerate(st["host"]):
        # pages in front of the first token that any row sees are not looked at
        first = max(0, length - n + 1 - case["window"]) // page if case["window"] else 0
        pages = st["block_table"][i, first:-(-length // page)].long()
        kv = []
        for cache in (st["k_cache"], st["v_cache"]):
            got = cache[pages].float()
            got = got.transpose(0, 1).flatten(1, 2) if case["heads_first"] else got.permute(2, 0, 1, 3).flatten(1, 2)
            kv.append(got[:, :length - first * page])
        k, v = kv                                                    # [key head][token][value]
        at = torch.arange(first * page, length, device="cuda")
        step = max(1, (1 << 27) // (hkv * g * at.shape[0]))
        for a in range(0, n, step):
            m = min(step, n - a)
            q = st["q"][start + a:start + a + m].float().view(m, hkv, g, d) * d ** -0.5
            s = torch.matmul(q.permute(1, 0, 2, 3).reshape(hkv, m * g, d), k.transpose(1, 2)).view(hkv, m, g, -1)
            where = torch.arange(length - n + a, length - n + a + m, device="cuda")[:, None]
            hidden = at > where
            if case["window"]:
                hidden = hidden | (at <= where - case["window"])
            s = s.masked_fill(hidden[None, :, None], -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(hkv, m * g, -1), v).view(hkv, m, g, d)
            out[start + a:start + a + m] = o.permute(1, 0, 2, 3).reshape(m, hkv * g, d).to(out.dtype)
    return out


def _plain_norm(case, st):
    x = st["x"].float()
    if case["post"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * st["post_weight"]
    if st["gate"] is not None:
        x = x * st["gate"].float()
    h = st["residual"].float() + st["scale"] * x
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * st["weight"]
    return h.to(st["residual"].dtype), y.to(st["x"].dtype)


def _plain_logprobs(case, st):
    v, top, every = case["v"], case["top"], []
    index = torch.arange(v, device="cuda")
    rows = max(1, (1 << 26) // v)
    for a in range(0, case["t"], rows):
        raw, target = st["logits"][a:a + rows].float(), st["targets"][a:a + rows].long()[:, None]
        mine = raw.gather(1, target)
        rank = 1 + (raw > mine).sum(1) + ((raw == mine) & (index < target)).sum(1)
        x = raw * case["scale"]
        x = x - x.amax(1, keepdim=True)
        e = torch.exp(x)
        total = e.sum(1, keepdim=True)
        lp = x.gather(1, target) - total.log()
        entropy = total.log()[:, 0] - (e * x.clamp_min(-1e30)).sum(1) / total[:, 0]
        got = [lp[:, 0], rank.to(torch.int32), entropy]
        if top:
            # the value's order as a whole number above the index's, so that no two are the same
            bits = (raw + 0.0).view(torch.int32).long()
            key = (torch.where(bits < 0, bits ^ 0x7fffffff, bits) << 32) | (v - 1 - index)
            best = v - 1 - (key.topk(top, 1).values & 0xffffffff)
            got += [best.to(torch.int32), x.gather(1, best) - total.log()]
        every.append(got)
    return tuple(torch.cat(one) for one in zip(*every))


# ---------------------------------------------------------------------------------------------------
# The framework's calls.  A program fills an operator's parameters once for the buffers it keeps, and launches.
# ---------------------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_chunk(case, st, keep):
    from paella_b200 import capi
    L, q, out, kc, table = capi.load(), st["q"], st["out"], st["k_cache"], st["block_table"]
    token, head = (kc.stride(2), kc.stride(1)) if case["heads_first"] else (kc.stride(1), kc.stride(2))
    p = capi.ChunkAttnParams(dtype=CODES[case["dtype"]], batch=case["b"], tokens=q.shape[0], q_heads=q.shape[1], kv_heads=case["hkv"],
                             head_dim=case["d"], page_size=case["page"], max_blocks=table.shape[1], max_new=case["new"],
                             max_len=st["max_len"], window=case["window"], scale=case["d"] ** -0.5, n_pages=kc.shape[0],
                             q_stride=q.stride(0), q_head_stride=q.stride(1), out_stride=out.stride(0), out_head_stride=out.stride(1),
                             page_stride=kc.stride(0), token_stride=token, head_stride=head, table_stride=table.stride(0), q=_ptr(q),
                             out=_ptr(out), k_cache=_ptr(kc), v_cache=_ptr(st["v_cache"]), block_table=_ptr(table),
                             starts=_ptr(st["starts"]), lens=_ptr(st["lens"]))
    info = capi.LaunchInfo()
    capi.check(L.pb_chunk_attn_info(C.byref(p), C.byref(info)), "pb_chunk_attn_info")
    scratch = torch.empty(max(16, info.scratch_bytes), dtype=torch.uint8, device="cuda")
    p.scratch, p.scratch_bytes = _ptr(scratch), info.scratch_bytes
    keep.update(launch=L.pb_chunk_attn_launch, params=p, out=out, buffers=scratch)


def _own_norm(case, st, keep):
    from paella_b200 import capi
    L, x, residual, gate = capi.load(), st["x"], st["residual"], st["gate"]
    h, y = torch.empty_like(residual), torch.empty_like(x)
    stream = "f32" if case["stream"] == "f32" else case["dtype"]
    p = capi.ResidualNormParams(tokens=case["t"], channels=case["c"], dtype=CODES[case["dtype"]], h_dtype=CODES[stream], scale=st["scale"],
                                eps=EPS, x_stride=x.stride(0), gate_stride=gate.stride(0) if case["gate"] == "token" else 0,
                                residual_stride=residual.stride(0), h_stride=h.stride(0), y_stride=y.stride(0), x=_ptr(x),
                                post_weight=_ptr(st["post_weight"]), gate=_ptr(gate), residual=_ptr(residual), h=_ptr(h),
                                weight=_ptr(st["weight"]), y=_ptr(y))
    keep.update(launch=L.pb_residual_norm_launch, params=p, out=(h, y))


def _own_logprobs(case, st, keep):
    from paella_b200 import capi
    L, t, top, logits = capi.load(), case["t"], case["top"], st["logits"]
    lp, entropy = torch.empty(t, device="cuda"), torch.empty(t, device="cuda")
    ranks = torch.empty(t, dtype=torch.int32, device="cuda")
    ids = torch.empty(t, top, dtype=torch.int32, device="cuda") if top else None
    lps = torch.empty(t, top, device="cuda") if top else None
    p = capi.LogprobsParams(tokens=t, vocab=case["v"], dtype=CODES[case["dtype"]], top=top, scale=case["scale"], logits_stride=logits.stride(0),
                            top_stride=top, logits=_ptr(logits), targets=_ptr(st["targets"]), logprobs=_ptr(lp), ranks=_ptr(ranks),
                            entropy=_ptr(entropy), top_ids=_ptr(ids), top_logprobs=_ptr(lps))
    keep.update(launch=L.pb_logprobs_launch, params=p, out=(lp, ranks, entropy, ids, lps) if top else (lp, ranks, entropy))


def run(st):
    case = st["case"]
    if own:
        keep = st["keep"]
        if not keep:
            {"chunk": _own_chunk, "norm": _own_norm, "logprobs": _own_logprobs}[case["op"]](case, st, keep)
        rc = keep["launch"](C.byref(keep["params"]), torch.cuda.current_stream().cuda_stream, 0, None)
        if rc != 0:
            from paella_b200 import capi
            capi.check(rc, keep["launch"].__name__)
        return keep["out"]
    return {"chunk": _plain_chunk, "norm": _plain_norm, "logprobs": _plain_logprobs}[case["op"]](case, st)


# ---------------------------------------------------------------------------------------------------
# What a pass cannot do without, and what it comes to in 64 bits
# ---------------------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "chunk":
        seen = read = 0
        for n, ctx in _lengths(case):
            w = case["window"] or n + ctx
            whole = min(n, max(0, w - ctx - 1))                      # rows whose window reaches the first token
            seen += whole * ctx + whole * (whole + 1) // 2 + (n - whole) * w
            read += min(n + ctx, n - 1 + w)
        es, d, new = BYTES[case["dtype"]], case["d"], sum(n for n, _ in _lengths(case))
        return {"bytes": 2 * es * d * case["hkv"] * (read + new * case["g"]) + 8 * case["b"] + 4 * (read // case["page"]),
                "flops": 4 * d * case["hkv"] * case["g"] * seen}
    if case["op"] == "norm":
        t, c, es = case["t"], case["c"], BYTES[case["dtype"]]
        stream = 4 if case["stream"] == "f32" else es
        gates = {"none": 0, "channel": c, "token": t * c}[case["gate"]]
        return {"bytes": 2 * t * c * (es + stream) + gates * es + 4 * c * (2 if case["post"] else 1),
                "flops": t * c * (6 + (4 if case["post"] else 0) + (1 if gates else 0))}
    t, v = case["t"], case["v"]
    return {"bytes": t * v * BYTES[case["dtype"]] + t * (16 + 8 * case["top"]), "flops": 6 * t * v}


def _exact_chunk(case, st):
    """head by head, with the whole of a sequence's scores"""
    hkv, g, d, page = case["hkv"], case["g"], case["d"], case["page"]
    out = st["out"].double()
    for i, (start, n, length) in enumerate(st["host"]):
        low = max(0, length - n + 1 - case["window"]) if case["window"] else 0
        at = torch.arange(low, length, device="cuda")
        pages, row = st["block_table"][i].long()[at // page], at % page
        k, v = ((c[pages, :, row] if case["heads_first"] else c[pages, row]) for c in (st["k_cache"], st["v_cache"]))
        behind = torch.arange(length - n, length, device="cuda")[:, None] - at      # how far a row's own token lies behind
        seen = behind >= 0
        if case["window"]:
            seen &= behind < case["window"]
        for h in range(hkv * g):
            keys, values = k[:, h // g].double(), v[:, h // g].double()
            for a in range(0, n, 1024):
                z = st["q"][start + a:start + min(n, a + 1024), h].double() @ keys.t() / math.sqrt(d)
                z = torch.where(seen[a:a + 1024], z, -math.inf)
                out[start + a:start + min(n, a + 1024), h] = torch.softmax(z, 1) @ values
    return out


def _exact_logprobs(case, st):
    every = []
    for t in range(0, case["t"], 256):
        raw, target = st["logits"][t:t + 256].double(), st["targets"][t:t + 256].long()
        lp = torch.log_softmax(raw * case["scale"], 1)
        entropy = -torch.special.xlogy(lp.exp(), lp.exp()).sum(1)
        order = torch.sort(raw, dim=1, descending=True, stable=True).indices
        rank = (order == target[:, None]).int().argmax(1) + 1
        got = [lp[torch.arange(len(target)), target], rank.to(torch.int32), entropy]
        if case["top"]:
            best = order[:, :case["top"]]
            got += [best.to(torch.int32), torch.take_along_dim(lp, best, 1)]
        every.append(got)
    return tuple(torch.cat(one) for one in zip(*every))


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "chunk":
        return _exact_chunk(case, st)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, st)
    h, y = [], []
    for t in range(0, case["t"], 4096):
        rows = slice(t, t + 4096)
        z = st["x"][rows].double()
        if case["post"]:
            z = z / (z.pow(2).sum(1, keepdim=True) / case["c"] + EPS).sqrt() * st["post_weight"].double()
        if case["gate"] != "none":
            z = torch.mul(z, st["gate"][rows if case["gate"] == "token" else slice(None)].double())
        z = torch.add(st["residual"][rows].double(), z, alpha=st["scale"])
        h.append(z)
        y.append(z / (z.pow(2).sum(1, keepdim=True) / case["c"] + EPS).sqrt() * st["weight"].double())
    return torch.cat(h), torch.cat(y)
