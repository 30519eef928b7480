"""Rotary positions, the 8-bit K/V cache and page-sparse attention: the cases they are measured on, their plain
forms in elementary torch operations, and their values in 64 bits.

Sizes come from the framework's own workloads (32 query / 8 KV heads of 128, 64 sequences of 1-8 k tokens; 24 query / 4 KV
heads of 256 with 64 rotated dims) and from what long-context serving does around them."""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---- the cases ----------------------------------------------------------------------------------------------------------
def _rope(name, tokens, hq, hkv, d, rot, dtype, layout, scaling, factor, context, inverse, fused):
    return dict(name=name, op="rope", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, dtype=dtype, layout=layout, scaling=scaling,
                factor=factor, context=context, inverse=inverse, fused=fused)


def _cache(name, op, n_seq, lo, hi, hq, hkv, d, page, dtype, **more):
    return dict(name=name, op=op, n_seq=n_seq, lo=lo, hi=hi, hq=hq, hkv=hkv, d=d, page=page, dtype=dtype, **more)


def listed():
    return [
        # one token of each of 64 sequences, q and k cut out of one projection's output rows
        _rope("rope_step", 64, 32, 8, 128, 128, "bf16", "halves", "none", 1.0, 32768, False, True),
        # a prefill chunk at far positions, a quarter of the head rotated, neighbours paired, context stretched 8 times
        _rope("rope_chunk_far", 8192, 24, 4, 256, 64, "f16", "pairs", "ramp", 8.0, 1000000, False, True),
        # the gradients of q and k over a packed batch of training sequences
        _rope("rope_gradient", 32768, 32, 8, 128, 128, "bf16", "halves", "bands", 8.0, 65536, True, False),
        # a prefill chunk written in 8 bits and read back flat, as prefix store and restore do
        _cache("q8_write_read", "q8_copy", 1, 4097, 4097, 32, 8, 128, 16, "bf16"),
        _cache("q8_write_read_wide", "q8_copy", 1, 30001, 30001, 24, 4, 256, 32, "f16"),
        # single-stream decode step (append of the token and attention), a short and a long context
        _cache("q8_step_short", "q8_step", 1, 1500, 1500, 24, 4, 256, 16, "bf16"),
        _cache("q8_step_long", "q8_step", 1, 131001, 131001, 32, 8, 128, 16, "f16"),
        # batched decode step over ragged sequences
        _cache("q8_step_batch", "q8_step", 64, 1024, 8192, 32, 8, 128, 16, "bf16"),
        # a prefill chunk attending to the 8-bit cache behind it
        _cache("q8_prefill", "q8_prefill", 1, 16384, 16384, 32, 8, 128, 16, "bf16", chunk=2048),
        # page-sparse decode: single stream, batch, and over the 8-bit cache
        _cache("sparse_stream", "sparse", 1, 32768, 32768, 24, 4, 256, 16, "bf16", top=64, first=1, last=4, pool="16"),
        _cache("sparse_batch", "sparse", 32, 8000, 32768, 32, 8, 128, 16, "bf16", top=128, first=1, last=8, pool="16"),
        _cache("sparse_q8", "sparse", 16, 30000, 65536, 32, 4, 128, 64, "f16", top=48, first=1, last=2, pool="e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hkv, group, d = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 6, 8, 12, 16]), rng.choice([64, 128, 256])
    dtype, page = rng.choice(["bf16", "f16"]), rng.choice([16, 32, 48, 64, 128])
    op = rng.choice(["rope", "q8_copy", "q8_step", "q8_step", "q8_prefill", "sparse", "sparse"])
    if op == "rope":
        while hkv * (group + 1) * d > 9216:
            hkv, group = max(1, hkv // 2), max(1, group // 2)
        rot = rng.choice([d, d // 2, d // 4, 2 * rng.randint(4, d // 2)])
        tokens = _log(rng, 1, 18000)
        scaling = rng.choice(["none", "linear", "base", "bands", "ramp"])
        return _rope("", tokens, hkv * group, hkv, d, rot, dtype, rng.choice(["halves", "pairs"]), scaling,
                     rng.choice([2.0, 4.0, 8.0, 20.0]), _log(rng, tokens + 1000, 1000000), rng.random() < 0.4, rng.random() < 0.5)
    if op == "q8_copy":
        n = _log(rng, 1, 50000000 // (hkv * d))
        return _cache("", op, 1, n, n, hkv * group, hkv, d, page, dtype)
    if op == "q8_prefill":
        group = min(group, 48 // hkv)
        depth = _log(rng, 1, 16384 * 4096 // max(4096, hkv * group * d))
        return _cache("", op, 1, depth, depth, hkv * group, hkv, d, page, dtype, chunk=min(depth, _log(rng, 1, 2048)))
    n_seq = _log(rng, 1, 64)
    cap = (290000000 if op == "q8_step" else 400000000) // (hkv * d * n_seq)
    hi = _log(rng, 300 if op == "sparse" else 1, min(cap, 131072 if op == "q8_step" else 100000))
    lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
    if op == "q8_step":
        return _cache("", op, n_seq, lo, hi, hkv * group, hkv, d, page, dtype)
    pages = -(-hi // page)
    top = max(4, min(_log(rng, 4, 256), pages // 4 + 4))
    return _cache("", op, n_seq, lo, hi, hkv * group, hkv, d, page, dtype, top=top, first=rng.choice([0, 1, 1, 2]),
                  last=rng.choice([1, 1, 2]), pool=rng.choice(["16", "e4m3"]))


def _lengths(case):
    """The sequences' lengths: from the case alone, the longest among them."""
    rng = random.Random(case["n_seq"] * 1000003 + case["lo"] * 31 + case["hi"])
    return [case["hi"]] + [rng.randint(case["lo"], case["hi"]) for _ in range(case["n_seq"] - 1)]


def work(case):
    if case["op"] == "rope":
        elems = case["tokens"] * (case["hq"] + case["hkv"])
        return {"bytes": elems * case["d"] * 4 + 4 * case["tokens"], "flops": elems * case["rot"] * 3}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    lens, n = _lengths(case), case["n_seq"]
    q8_row = 2 * (d + 1) * hkv                       # K and V of one token: 8 bits an element, one exponent a row
    if case["op"] == "q8_copy":                      # source, cache written, cache read, flat result
        return {"bytes": lens[0] * (2 * q8_row + 2 * 4 * d * hkv), "flops": lens[0] * 2 * d * hkv * 4}
    if case["op"] == "q8_step":
        new = n * (4 * hkv * d + q8_row + 4 * hq * d)
        return {"bytes": sum(lens) * q8_row + new, "flops": sum(lens) * hq * d * 4}
    if case["op"] == "q8_prefill":
        m, depth = case["chunk"], case["hi"]
        keys = m * depth - m * (m - 1) // 2
        return {"bytes": depth * q8_row + 4 * m * hq * d, "flops": keys * hq * d * 4}
    row = q8_row if case["pool"] == "e4m3" else 4 * d * hkv
    total = picked = 0
    for length in lens:
        pages = -(-length // case["page"])
        total += pages
        picked += length if pages <= case["top"] else (case["top"] - 1) * case["page"] + length - (pages - 1) * case["page"]
    return {"bytes": total * hkv * (2 * d + 1) + picked * row + n * (4 * hq * d + 4 * hkv * case["top"]),
            "flops": total * hq * d * 2 + picked * hq * d * 4}


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(case, seed):
    """What the model hands over: seeded, on the GPU."""
    g = _gen(seed)
    t = DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    if case["op"] == "rope":
        n = case["tokens"]
        if case["fused"]:
            rows = normal(n, (hq + 2 * hkv) * d).to(t)
            q = rows[:, :hq * d].unflatten(1, (hq, d))
            k = rows[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        else:
            q, k = normal(n, hq, d).to(t), normal(n, hkv, d).to(t)
        start = torch.randint(0, case["context"] - n + 1, (1,), generator=g, device="cuda", dtype=torch.int32)
        pos = start + torch.arange(n, device="cuda", dtype=torch.int32)
        return {"q": q, "k": k, "pos": pos.contiguous()}
    # keys have channels of unlike size and a common offset, as keys do; values differ in size from token to token
    spread = torch.exp(0.5 * normal(hkv, d))
    offset = normal(hkv, d) * spread
    ks, vs = [], []
    for length in _lengths(case):
        ks.append((normal(length, hkv, d) * spread + offset).to(t))
        vs.append((normal(length, hkv, d) * torch.exp(0.3 * normal(length, hkv, 1))).to(t))
    rows = case.get("chunk", 0) if case["op"] == "q8_prefill" else case["n_seq"]
    q = normal(rows, hkv, hq // hkv, d)
    if case["op"] == "sparse":                       # queries that look for something the sequence holds
        for b, k in enumerate(ks):
            at = torch.randint(0, k.shape[0], (hkv,), generator=g, device="cuda")
            q[b] += 0.5 * (k[at, torch.arange(hkv, device="cuda")].float() - offset)[:, None, :]
    return {"k": ks, "v": vs, "q": q.reshape(rows, hq, d).to(t).contiguous()}


# ---- plain forms: the 8-bit cache ---------------------------------------------------------------------------------------
def _times_power(x, e):
    """x * 2^e, exact: the power is put together from its bits."""
    return (x.double() * ((e.long() + 1023) << 52).view(torch.float64)).float()


def _quantise(x):
    """Rows of 8-bit values and one power of two each: e the smallest integer with max|x| <= 448 * 2^e."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    mant, exp = torch.frexp(amax)                    # amax = mant * 2^exp, mant in [1/2, 1)
    e = torch.where(mant <= 0.875, exp - 9, exp - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(-127, 120)
    return _times_power(x, -e).to(torch.float8_e4m3fn), e


def _expand(q8, e):
    return _times_power(q8.float(), e)


def _attend(q, k, v, scale, first_visible=None):
    """q [rows, hq, d], k and v [keys, hkv, d] in 32 bits; row r sees keys up to first_visible + r (None: all)."""
    rows, hq, d = q.shape
    keys, hkv, _ = k.shape
    out = torch.empty(rows, hq, d, device=q.device, dtype=torch.float32)
    g = hq // hkv
    step = max(1, 200000000 // (rows * keys * g))
    for h in range(0, hkv, step):
        n = min(step, hkv - h)
        qh = q[:, h * g:(h + n) * g].reshape(rows, n, g, d).permute(1, 2, 0, 3).reshape(n, g * rows, d)
        s = torch.matmul(qh, k[:, h:h + n].permute(1, 2, 0)) * scale
        if first_visible is not None:
            hidden = torch.arange(keys, device=q.device)[None, :] > first_visible + torch.arange(rows, device=q.device)[:, None]
            s = s.reshape(n, g, rows, keys).masked_fill(hidden, float("-inf")).reshape(n, g * rows, keys)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p, v[:, h:h + n].permute(1, 0, 2)) / p.sum(-1, keepdim=True)
        out[:, h * g:(h + n) * g] = o.reshape(n, g, rows, d).permute(2, 0, 1, 3).reshape(rows, n * g, d)
    return out


# ---- plain forms: page bounds and selection -----------------------------------------------------------------------------
def _pages(x, page, fill):
    n = -(-x.shape[0] // page)
    pad = torch.full((n * page - x.shape[0], *x.shape[1:]), fill, device=x.device, dtype=x.dtype)
    return torch.cat([x, pad]).unflatten(0, (n, page))


def _int8_exponent(amax):
    mant, exp = torch.frexp(amax)
    return torch.where(amax > 0, torch.where(mant <= 127 / 128, exp - 7, exp - 6), torch.full_like(exp, -126)).clamp(-126, 121)


def _bounds(k, page):
    """Largest and smallest key of every page's channels, rounded outwards to 8-bit whole numbers of 2^e."""
    k = k.float()
    top, bottom = _pages(k, page, float("-inf")).amax(1), _pages(k, page, float("inf")).amin(1)   # [pages, hkv, d]
    e = _int8_exponent(torch.maximum(top.abs(), bottom.abs()).amax(-1, keepdim=True))
    return torch.ceil(_times_power(top, -e)), torch.floor(_times_power(bottom, -e)), e[..., 0]


def _select(q, top_b, bottom_b, e, case):
    """Pages of one sequence, per KV head: q [hq, d]; ascending, padded with -1 to case["top"]."""
    hkv, top = case["hkv"], case["top"]
    n = top_b.shape[0]
    qf = q.float().reshape(hkv, -1, q.shape[-1])
    f = _int8_exponent(qf.abs().amax(-1, keepdim=True))
    q8 = torch.round(_times_power(qf, -f))
    up, down = q8.clamp(min=0), q8.clamp(max=0)
    # whole numbers below 2^22: exact in 32 bits
    s = torch.einsum("hgd,phd->hgp", up, top_b) + torch.einsum("hgd,phd->hgp", down, bottom_b)
    s = _times_power(s, f + e.t()[:, None, :]).amax(1)                                             # [hkv, pages]
    index = torch.arange(n, device=q.device)
    s = s.masked_fill((index < case["first"]) | (index >= n - case["last"]), float("inf"))
    best = torch.sort(s, dim=-1, descending=True, stable=True).indices[:, :min(top, n)].sort(-1).values
    return torch.nn.functional.pad(best, (0, top - best.shape[1]), value=-1).int()


def _attend_pages(q, k, v, sel, page, scale):
    """One row: q [hq, d] over the listed pages of every KV head, k and v [keys, hkv, d] in 32 bits."""
    hkv = k.shape[1]
    keys = (sel.long()[:, :, None] * page + torch.arange(page, device=q.device)).flatten(1)       # [hkv, slots]
    live = (sel >= 0).repeat_interleave(page, 1) & (keys < k.shape[0])
    keys = keys.clamp(0, k.shape[0] - 1)
    heads = torch.arange(hkv, device=q.device)[:, None]
    s = torch.matmul(q.reshape(hkv, -1, q.shape[-1]), k[keys, heads].transpose(1, 2)) * scale
    s = s.masked_fill(~live[:, None, :], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return (torch.matmul(p, v[keys, heads]) / p.sum(-1, keepdim=True)).reshape(q.shape)


# ---- plain form: rotary positions ---------------------------------------------------------------------------------------
THETA = 1.0e6
ORIGINAL = 8192


def _frequencies(case, pairs):
    """Radians a position, per pair, in 64 bits."""
    rot, factor = case["rot"], case["factor"]
    theta = THETA * factor ** (rot / (rot - 2)) if case["scaling"] == "base" else THETA
    i = torch.arange(pairs, dtype=torch.float64, device="cuda")
    f = theta ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "bands":                 # long wavelengths divided, short ones kept, a blend between
        turns = ORIGINAL * f / (2 * math.pi)
        blend = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = f * ((1 - blend) / factor + blend)
    elif case["scaling"] == "ramp":                  # a linear ramp over the pairs between 32 turns and 1
        def pair_of(turns):
            return rot * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), rot - 1)
        r = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / factor * r + f * (1 - r)
    return f


def _rope_factor(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "ramp" else 1.0


def _rotate(x, cos, sin, case):
    rot = case["rot"]
    xf = x.float()
    if case["layout"] == "halves":
        a, b = xf[..., :rot // 2], xf[..., rot // 2:rot]
    else:
        a, b = xf[..., 0:rot:2], xf[..., 1:rot:2]
    ya, yb = a * cos - b * sin, b * cos + a * sin
    y = xf.clone()
    if case["layout"] == "halves":
        y[..., :rot // 2], y[..., rot // 2:rot] = ya, yb
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = ya, yb
    return y.to(x.dtype)


# ---- the framework's side: what a user's program keeps -------------------------------------------------------------------
def _stream():
    return torch.cuda.current_stream()


def _engine(case, x, cached, seed):
    """An engine whose cache holds the first cached[b] tokens of every sequence, pages scattered over the pool."""
    from deusridet_b200 import PagedKVEngine
    lens = _lengths(case)
    need = [-(-n // case["page"]) for n in lens]
    eng = PagedKVEngine(num_layers=1, num_q_heads=case["hq"], num_kv_heads=case["hkv"], head_dim=case["d"], page_size=case["page"],
                        dtype=case["dtype"], kv_dtype="e4m3" if case.get("pool", "e4m3") == "e4m3" else None, rotary_dim=0,
                        max_pages=max(4, sum(need)), max_seqs=case["n_seq"], max_pages_per_seq=max(need), device=0)
    if case["op"] == "sparse":
        eng.page_bounds_enable()
    pages = [eng.alloc_block() for _ in range(max(4, sum(need)))]
    random.Random(seed).shuffle(pages)
    for p in pages:
        eng.free_block(p)
    seqs = []
    for b, n in enumerate(lens):
        s = eng.seq_create()
        assert eng.ensure_blocks_for_range(s, 0, n, _stream())
        eng.set_seq_len(s, n)
        seqs.append(s)
    eng.sync_block_table(_stream())
    for b, s in enumerate(seqs):
        if cached[b] > 0:
            eng.append_rope_chunk(0, s, 0, cached[b], x["k"][b][:cached[b]].contiguous(), x["v"][b][:cached[b]].contiguous(),
                                  _stream())
    return eng, seqs


def prepare(case, seed):
    x = _inputs(case, seed)
    st = {"case": case, "x": x}
    if case["op"] == "rope":
        if own:
            from deusridet_b200 import Rope
            kw = {"none": {}, "linear": dict(factor=case["factor"]), "base": dict(factor=case["factor"]),
                  "bands": dict(factor=case["factor"], original_context=ORIGINAL, low_freq_factor=1.0, high_freq_factor=4.0),
                  "ramp": dict(factor=case["factor"], original_context=ORIGINAL, beta_fast=32.0, beta_slow=1.0)}[case["scaling"]]
            st["rope"] = Rope(head_dim=case["d"], rotary_dim=case["rot"], theta=THETA, layout=case["layout"], dtype=case["dtype"],
                              scaling=case["scaling"], device=0, **kw)
            st["q_out"] = torch.empty(x["q"].shape, device="cuda", dtype=x["q"].dtype)
            st["k_out"] = torch.empty(x["k"].shape, device="cuda", dtype=x["k"].dtype)
        return st
    lens, d, op = _lengths(case), case["d"], case["op"]
    st["scale"] = 1.0 / math.sqrt(d)
    if op == "q8_step":                              # the step brings every sequence's last token
        st["k_new"] = torch.stack([k[-1] for k in x["k"]])
        st["v_new"] = torch.stack([v[-1] for v in x["v"]])
    if own:
        cached = [0 if op == "q8_copy" else n - 1 if op == "q8_step" else n for n in lens]
        st["eng"], st["seqs"] = _engine(case, x, cached, seed)
        st["rows"] = torch.tensor(st["seqs"], device="cuda", dtype=torch.int32)
        st["lens"] = torch.tensor(lens, device="cuda", dtype=torch.int32)
        st["out"] = torch.zeros_like(x["q"])
        if op == "q8_copy":
            st["flat"] = torch.empty(1, 2, lens[0], case["hkv"], d, device="cuda", dtype=x["q"].dtype)
        if op == "sparse":
            st["sel"] = torch.empty(case["n_seq"], case["hkv"], case["top"], device="cuda", dtype=torch.int32)
        torch.cuda.synchronize()
    elif op in ("q8_step", "q8_prefill") or case.get("pool") == "e4m3":
        st["kq"], st["vq"] = [_quantise(k) for k in x["k"]], [_quantise(v) for v in x["v"]]
    if op == "sparse" and not own:
        ks = [_expand(*k) for k in st["kq"]] if case["pool"] == "e4m3" else x["k"]
        st["bounds"] = [_bounds(k, case["page"]) for k in ks]
    return st


def run(st):
    case, x = st["case"], st["x"]
    return (_run_own if own else _run_plain)(case, x, st)


def _run_own(case, x, st):
    if case["op"] == "rope":
        st["rope"].apply(x["pos"], x["q"], x["k"], out_q=st["q_out"], out_k=st["k_out"], inverse=case["inverse"], stream=_stream())
        return st["q_out"], st["k_out"]
    eng, hi = st["eng"], case["hi"]
    if case["op"] == "q8_copy":
        eng.append_rope_chunk(0, st["seqs"][0], 0, hi, x["k"][0], x["v"][0], _stream())
        eng.extract(st["seqs"][0], 0, hi, st["flat"], _stream())
        return st["flat"]
    if case["op"] == "q8_step":
        eng.append_attend_decode(0, case["n_seq"], st["rows"], st["lens"], hi, st["k_new"], st["v_new"], x["q"], st["out"],
                                 st["scale"], _stream())
        return st["out"]
    if case["op"] == "q8_prefill":
        eng.attend_prefill_chunk(0, st["seqs"][0], hi - case["chunk"], case["chunk"], x["q"], st["out"], st["scale"], _stream())
        return st["out"]
    eng.select_pages(0, case["n_seq"], st["rows"], st["lens"], hi, x["q"], case["top"], case["first"], case["last"], st["sel"],
                     _stream())
    eng.attend_selected(0, case["n_seq"], st["rows"], st["lens"], hi, st["sel"], case["top"], x["q"], st["out"], st["scale"],
                        _stream())
    return st["out"], st["sel"]


def _run_plain(case, x, st):
    t = DTYPES[case["dtype"]]
    if case["op"] == "rope":
        angle = x["pos"].double()[:, None] * _frequencies(case, case["rot"] // 2)[None, :]
        cos = (_rope_factor(case) * torch.cos(angle)).float()[:, None, :]
        sin = (_rope_factor(case) * torch.sin(angle)).float()[:, None, :]
        if case["inverse"]:
            sin = -sin
        return _rotate(x["q"], cos, sin, case), _rotate(x["k"], cos, sin, case)
    if case["op"] == "q8_copy":
        return torch.stack([_expand(*_quantise(y[0])) for y in (x["k"], x["v"])])[None].to(t)
    if case["op"] == "q8_prefill":
        k, v = _expand(*st["kq"][0]), _expand(*st["vq"][0])
        return _attend(x["q"].float(), k, v, st["scale"], case["hi"] - case["chunk"]).to(t)
    out, sel = [], []
    for b in range(case["n_seq"]):
        if case["op"] == "q8_step":                  # the token is quantised and written into its place, then attended to
            for cache, new in ((st["kq"], st["k_new"]), (st["vq"], st["v_new"])):
                q8, e = _quantise(new[b])
                cache[b][0].view(torch.uint8)[-1], cache[b][1][-1] = q8.view(torch.uint8), e
            out.append(_attend(x["q"][b:b + 1].float(), _expand(*st["kq"][b]), _expand(*st["vq"][b]), st["scale"])[0])
        else:
            sel.append(_select(x["q"][b], *st["bounds"][b], case))
            if case["pool"] == "e4m3":
                k, v = _expand(*st["kq"][b]), _expand(*st["vq"][b])
            else:
                k, v = x["k"][b].float(), x["v"][b].float()
            out.append(_attend_pages(x["q"][b].float(), k, v, sel[-1], case["page"], st["scale"]))
    out = torch.stack(out).to(t)
    return (out, torch.stack(sel)) if sel else out


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def _power(e):
    """2^e for whole numbers e held in 64 bits; a table, because a power function need not be exact."""
    table = torch.tensor([2.0 ** i for i in range(-400, 401)], dtype=torch.float64, device="cuda")
    return table[(e + 400).long()]


def _exact_stored(x):
    """The values an 8-bit row stands for: 3 mantissa bits below the leading one, ties to even, steps of 2^-9 at least."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -150) / 448.0))
    e = torch.where(448.0 * _power(e - 1) >= amax, e - 1, e)      # the logarithm may be off by one at a border
    e = torch.where(448.0 * _power(e) < amax, e + 1, e)
    e = e.clamp(-127, 120)
    y = x * _power(-e)
    lead = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    lead = torch.where(_power(lead) > y.abs().clamp(min=2.0 ** -6), lead - 1, lead)
    step = _power(lead - 3)
    return torch.round(y / step) * step * _power(e)


def _exact_softmax_sum(q, k, v, scale):
    """q [n, d], k and v [keys, d] in 64 bits."""
    return torch.softmax((q @ k.T) * scale, -1) @ v


def _exact_sparse(case, x, b):
    page, hq, hkv, d = case["page"], case["hq"], case["hkv"], case["d"]
    g, scale = hq // hkv, 1.0 / math.sqrt(d)
    k, v = x["k"][b].double(), x["v"][b].double()
    if case["pool"] == "e4m3":
        k, v = _exact_stored(k), _exact_stored(v)
    n = -(-k.shape[0] // page)
    owner = torch.arange(k.shape[0], device="cuda") // page
    out = torch.empty(hq, d, dtype=torch.float64, device="cuda")
    sel = torch.full((hkv, case["top"]), -1, dtype=torch.int32, device="cuda")

    def whole(y, exact_top):                         # smallest 2^e with |y| <= 127 * 2^e
        e = torch.ceil(torch.log2(exact_top.clamp(min=2.0 ** -150) / 127.0))
        e = torch.where(127.0 * _power(e - 1) >= exact_top, e - 1, e)
        e = torch.where(127.0 * _power(e) < exact_top, e + 1, e).clamp(-126, 121)
        return _power(e)

    for h in range(hkv):
        at = owner[:, None].expand(-1, d)
        hi = torch.full((n, d), -math.inf, dtype=torch.float64, device="cuda").scatter_reduce(0, at, k[:, h], "amax")
        lo = torch.full((n, d), math.inf, dtype=torch.float64, device="cuda").scatter_reduce(0, at, k[:, h], "amin")
        unit = whole(hi, torch.maximum(hi.abs(), lo.abs()).amax(1, keepdim=True))
        hi, lo = torch.ceil(hi / unit) * unit, torch.floor(lo / unit) * unit
        qh = x["q"][b, h * g:(h + 1) * g].double()
        q_unit = whole(qh, qh.abs().amax(1, keepdim=True))
        q8 = torch.round(qh / q_unit) * q_unit
        bound = torch.full((n,), -math.inf, dtype=torch.float64, device="cuda")
        for r in range(g):
            bound = torch.maximum(bound, torch.maximum(q8[r] * hi, q8[r] * lo).sum(1))
        must = set(range(min(case["first"], n))) | set(range(max(0, n - case["last"]), n))
        value = bound.tolist()
        order = sorted(range(n), key=lambda p: (p not in must, -value[p], p))
        pick = sorted(order[:min(case["top"], n)])
        sel[h, :len(pick)] = torch.tensor(pick, dtype=torch.int32, device="cuda")
        rows = torch.isin(owner, torch.tensor(pick, device="cuda"))
        out[h * g:(h + 1) * g] = _exact_softmax_sum(qh, k[rows, h], v[rows, h], scale)
    return out, sel


def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "rope":
        rot, half = case["rot"], case["rot"] // 2
        f = _frequencies(case, half)
        angle = torch.outer(x["pos"].double(), f)
        turn = torch.polar(torch.full_like(angle, _rope_factor(case)), -angle if case["inverse"] else angle)
        res = []
        for y in (x["q"], x["k"]):
            y = y.double()
            if case["layout"] == "halves":
                z = torch.complex(y[..., :half].contiguous(), y[..., half:rot].contiguous()) * turn[:, None, :]
                res.append(torch.cat([z.real, z.imag, y[..., rot:]], -1))
            else:
                z = torch.view_as_complex(y[..., :rot].unflatten(-1, (half, 2)).contiguous()) * turn[:, None, :]
                res.append(torch.cat([torch.view_as_real(z).flatten(-2), y[..., rot:]], -1))
        return tuple(res)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g, scale = hq // hkv, 1.0 / math.sqrt(d)
    if case["op"] == "q8_copy":
        return torch.stack([_exact_stored(x["k"][0]), _exact_stored(x["v"][0])])[None]
    if case["op"] == "q8_prefill":
        m, depth = case["chunk"], case["hi"]
        k, v = _exact_stored(x["k"][0]), _exact_stored(x["v"][0])
        out = torch.empty(m, hq, d, dtype=torch.float64, device="cuda")
        for h in range(hq):
            for t0 in range(0, m, 512):
                t1 = min(m, t0 + 512)
                n = depth - m + t1
                s = (x["q"][t0:t1, h].double() @ k[:n, h // g].T) * scale
                s += torch.triu(torch.full_like(s, -math.inf), diagonal=depth - m + t0 + 1)
                out[t0:t1, h] = torch.softmax(s, -1) @ v[:n, h // g]
        return out
    out, sel = [], []
    for b in range(case["n_seq"]):
        if case["op"] == "sparse":
            o, s = _exact_sparse(case, x, b)
            out.append(o)
            sel.append(s)
            continue
        k, v = _exact_stored(x["k"][b]), _exact_stored(x["v"][b])
        out.append(torch.cat([_exact_softmax_sum(x["q"][b, h * g:(h + 1) * g].double(), k[:, h], v[:, h], scale) for h in range(hkv)]))
    return (torch.stack(out), torch.stack(sel)) if sel else torch.stack(out)
