"""What is measured of the 4-bit ICL cache and the attention that reads it.

Three kinds of case, over the public entry points of the cache:

  store   irx_icl4_encode and irx_icl4_decode: keys and values of 64-wide heads
          into the 4-bit cache, and what it holds read back, with the blocks'
          bounds.
  attend  irx_icl4_attention: softmax(q k^T / 8) v over the cached rows, each
          estimator's own number of them, rows left out by a bit mask.
  choose  irx_icl4_select, then irx_icl4_attention over the blocks of 64 rows
          it picked for each query.

The cache's bytes are laid out as the library's header states; a state holds
them as a user's program does. Sizes are those of the benchmark's contexts
(1,024, 50,000 and 200,000 training rows) and of odd tables between.

torch is imported before the backend, so that both use one HIP runtime.
"""

import functools
import math

import torch

own = False

SCALE = 0.125  # 1 / sqrt(64)
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # what the codes 0..7 stand for; 8..15 are their negatives


def listed():
    return [
        # A small table's context, one ICL block: the call's own cost counts.
        {"name": "store_small", "kind": "store", "estimators": 1, "rows": 1024, "element": "f32", "layout": "heads",
         "ragged": False},
        # The benchmark's context, one ICL block.
        {"name": "store_context", "kind": "store", "estimators": 1, "rows": 50000, "element": "f32",
         "layout": "heads", "ragged": False},
        # Two estimators of different lengths as FP16 token rows, as a projection writes them.
        {"name": "store_ragged", "kind": "store", "estimators": 2, "rows": 12345, "element": "f16",
         "layout": "tokens", "ragged": True},
        # Serving one row against 50,000: the cache is read once.
        {"name": "attend_row", "kind": "attend", "estimators": 1, "rows": 50000, "queries": 1, "element": "f32",
         "layout": "heads", "ragged": False, "masked": False},
        # A few dozen rows over two small contexts: latency.
        {"name": "attend_small", "kind": "attend", "estimators": 2, "rows": 1024, "queries": 33, "element": "f32",
         "layout": "heads", "ragged": False, "masked": False},
        # Eight served rows over an ensemble of two 200,000-row contexts.
        {"name": "attend_serve", "kind": "attend", "estimators": 2, "rows": 200000, "queries": 8, "element": "f16",
         "layout": "tokens", "ragged": False, "masked": False},
        # One 512-row pass over the benchmark's context.
        {"name": "attend_pass", "kind": "attend", "estimators": 1, "rows": 50000, "queries": 512, "element": "f32",
         "layout": "heads", "ragged": False, "masked": False},
        # An odd pass over two contexts of different lengths with rows held out of them.
        {"name": "attend_masked", "kind": "attend", "estimators": 2, "rows": 12345, "queries": 777,
         "element": "f16", "layout": "tokens", "ragged": True, "masked": True},
        # As many queries as rows, as where a context attends to itself.
        {"name": "attend_self", "kind": "attend", "estimators": 1, "rows": 10007, "queries": 10007,
         "element": "f16", "layout": "heads", "ragged": False, "masked": False},
        # One served row over 200,000, the 64 best of 3,125 blocks.
        {"name": "choose_row", "kind": "choose", "estimators": 1, "rows": 200000, "queries": 1, "blocks": 64,
         "element": "f32", "layout": "heads", "ragged": False, "masked": False},
        # A 512-row pass over the benchmark's context, each row its 32 best of 782 blocks.
        {"name": "choose_pass", "kind": "choose", "estimators": 1, "rows": 50000, "queries": 512, "blocks": 32,
         "element": "f32", "layout": "heads", "ragged": False, "masked": False},
        # An odd batch, two contexts of different lengths, rows held out.
        {"name": "choose_masked", "kind": "choose", "estimators": 2, "rows": 12345, "queries": 77, "blocks": 17,
         "element": "f16", "layout": "tokens", "ragged": True, "masked": True},
    ]


# ---- draws ----

def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed kinds: sizes uniform in their logarithm, no dearer
    than the dearest listed one of its kind, in time and in what the plain
    form holds."""
    while True:
        kind = rng.choice(("store", "attend", "attend", "choose", "choose"))
        case = {"kind": kind, "estimators": rng.randint(1, 4), "rows": _log(rng, 60, 200000),
                "element": rng.choice(("f32", "f16")), "layout": rng.choice(("heads", "tokens")),
                "ragged": rng.random() < 0.4}
        if kind != "store":
            case["masked"] = rng.random() < 0.4
            case["queries"] = _log(rng, 1, 10007)
        if kind == "choose":
            case["blocks"] = _log(rng, 1, 128)
        if case["estimators"] * case["rows"] > 400000:
            continue
        if _held(case) <= max(_held(c) for c in listed() if c["kind"] == kind):
            return case


def _held(case):
    """Numbers that the plain form holds at once."""
    pairs = 8 * case["estimators"]
    if case["kind"] == "store":
        return pairs * case["rows"] * 64
    if case["kind"] == "attend":
        return pairs * case["rows"] * case["queries"]
    return pairs * case["queries"] * (case["blocks"] * 64 * 64 + case["rows"] // 64)


# ---- work ----

def work(case):
    e, n, q = case["estimators"], case["rows"], case.get("queries", 0)
    pairs, tiles, el = 8 * e, -(-n // 64), 2 if case["element"] == "f16" else 4
    if case["kind"] == "store":
        cache = pairs * (tiles * 4480 + 256)
        bounds = pairs * tiles * 2 * 64 * 4
        return {"bytes": float(4 * pairs * n * 64 * el + 2 * cache + bounds), "flops": 0.0}
    rows = pairs * q * (2 * 64 * el + 4)
    masks = e * tiles * 8 if case["masked"] else 0
    if case["kind"] == "attend":
        return {"bytes": float(pairs * tiles * 4352 + rows + masks), "flops": 4.0 * 64 * pairs * q * n}
    chosen = min(case["blocks"], tiles)
    read = min(tiles, q * chosen) * 4352 + tiles * 128
    return {"bytes": float(pairs * read + rows + 4 * pairs * q * case["blocks"] + masks),
            "flops": float(pairs * q) * (2 * 128 * tiles + 4 * 64 * 64 * chosen)}


# ---- inputs ----

def _type(case):
    return torch.float16 if case["element"] == "f16" else torch.float32


def _rows(case, g, rows):
    """[E, 8, rows, 64] standard normal, as one head after another or as views of token rows [E, rows, 512]."""
    e = case["estimators"]
    if case["layout"] == "tokens":
        return torch.randn(e, rows, 8, 64, generator=g, device="cuda").transpose(1, 2)
    return torch.randn(e, 8, rows, 64, generator=g, device="cuda")


def _sources(case, seed):
    """Keys, values, queries (or None), lengths and kept rows (or None). The
    keys' channels differ in size, as learned ones do, and rows that stand
    together are alike, as in a table sorted by one of its columns."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    e, n = case["estimators"], case["rows"]
    gain = torch.exp(0.5 * torch.randn(e, 8, 1, 64, generator=g, device="cuda"))
    steps = torch.randn(e, 8, -(-n // 48), 64, generator=g, device="cuda")
    near = torch.arange(n, device="cuda") // 48
    k = _rows(case, g, n).mul_(0.8).add_(steps[:, :, near], alpha=0.6).mul_(gain).to(_type(case))
    v = _rows(case, g, n).to(_type(case))
    q = None if case["kind"] == "store" else _rows(case, g, case["queries"]).mul_(1.5).to(_type(case))
    lengths = keep = None
    if case["ragged"]:
        lengths = torch.randint(n // 2, n + 1, (e,), generator=g, device="cuda", dtype=torch.int32)
        if e > 2:
            lengths[-1] = 0  # an estimator without rows
    if case.get("masked"):
        keep = torch.rand(e, n, generator=g, device="cuda") < 0.8
        keep &= torch.rand(e, -(-n // 200), generator=g, device="cuda")[:, torch.arange(n, device="cuda") // 200] < 0.9
    return k, v, q, lengths, keep


def _bits(keep):
    """[E, N] truth values as 64-bit words, row r at bit r % 64 of word r / 64."""
    e, n = keep.shape
    padded = torch.zeros(e, -(-n // 64) * 64, dtype=torch.int64, device=keep.device)
    padded[:, :n] = keep
    return (padded.view(e, -1, 64) << torch.arange(64, device=keep.device)).sum(-1)


def prepare(case, seed):
    k, v, q, lengths, keep = _sources(case, seed)
    shape = (case["estimators"], 8, case["rows"])
    if case["kind"] == "store":
        state = {"kind": "store", "shape": shape, "k": k, "v": v, "lengths": lengths}
    else:
        state = {"kind": case["kind"], "shape": shape, "q": q, "cache": _encoded(k, v, lengths), "lengths": lengths,
                 "keep": None if keep is None else _bits(keep), "blocks": case.get("blocks", 0)}
    torch.cuda.synchronize()
    return state


# ---- the plain forms ----

def _pow2(e):
    """2^e exactly, for whole -126..127."""
    return (e.int() + 127 << 23).view(torch.float32)


def _exponents(largest):
    """The smallest e with largest <= 6 * 2^e, held to -13..13."""
    part, power = torch.frexp(largest)
    return torch.where(part <= 0.75, power - 3, power - 2).masked_fill(largest == 0, -13).clamp(-13, 13)


def _codes(x, e):
    """E2M1 codes of x / 2^e, to nearest, ties to the even code, saturated."""
    m = x.abs() * _pow2(-e)
    code = (m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)
    return code + 8 * (x < 0).to(torch.uint8)


def _quantized(k, v, lengths):
    """Codes [P, T * 64, 64] and exponents of keys [P, T * 64, 2] and values
    [P, T * 2, 64]; rows past an estimator's length are zero."""
    e, h, n, _ = k.shape
    tiles = -(-n // 64)
    kp, vp = (torch.nn.functional.pad(x.float(), (0, 0, 0, tiles * 64 - n)) for x in (k, v))
    if lengths is not None:
        past = (torch.arange(tiles * 64, device=k.device) >= lengths[:, None])[:, None, :, None]
        kp, vp = kp.masked_fill(past, 0.0), vp.masked_fill(past, 0.0)
    kp, vp = kp.reshape(e * h, tiles * 64, 2, 32), vp.reshape(e * h, tiles * 2, 32, 64)
    ke, ve = _exponents(kp.abs().amax(-1)), _exponents(vp.abs().amax(2))
    return (_codes(kp, ke[..., None]).flatten(2), ke, _codes(vp, ve[:, :, None]).flatten(1, 2), ve)


def _bounds(k, n, lengths, heads):
    """Per block and dim the floor and ceiling of the smallest and largest key
    (values k [P, T * 64, 64]) in steps of 2^x, x per (pair, dim), and 2^x."""
    pairs, rows, _ = k.shape
    row = torch.arange(rows, device=k.device)
    inside = (row < n).expand(pairs, rows)
    if lengths is not None:
        inside = inside & (row < lengths.repeat_interleave(heads)[:, None])
    part, power = torch.frexp(k.abs().amax(1))  # rows past the length are zero
    x = torch.where(part <= 127.0 / 128.0, power - 7, power - 6).masked_fill(k.abs().amax(1) == 0, -20)
    inside = inside[..., None]
    low = k.masked_fill(~inside, math.inf).view(pairs, -1, 64, 64).amin(2)
    high = k.masked_fill(~inside, -math.inf).view(pairs, -1, 64, 64).amax(2)
    empty = ~inside.view(pairs, -1, 64).any(-1, keepdim=True)
    low, high = (b.masked_fill(empty, 0.0) * _pow2(-x[:, None]) for b in (low, high))
    return low.floor(), high.ceil(), _pow2(x)


def _values(codes, e):
    table = torch.tensor(LEVELS + tuple(-level for level in LEVELS), device=codes.device)
    return table[codes.long()] * _pow2(e)


def _encoded(k, v, lengths):
    """The cache's bytes: per (pair, block) the codes of keys and values in the
    order in which the matrix products read them, then their exponents; the
    bounds; their scales."""
    n, heads = k.shape[2], k.shape[1]
    kc, ke, vc, ve = _quantized(k, v, lengths)
    low, high, scales = _bounds(_values(kc, ke.repeat_interleave(32, dim=2)), n, lengths, heads)
    pairs = kc.shape[0]
    tiles = kc.shape[1] // 64
    # Key 32 s + 16 a + 8 b + i, dim 16 g + 2 y + z: byte [s][g][a][i][b][y], nibble z.
    kc = kc.view(pairs, tiles, 2, 2, 2, 8, 4, 8, 2).permute(0, 1, 2, 6, 3, 5, 4, 7, 8)
    # Key 32 s + 16 t + 8 b + 4 h + 2 y + z, dim 16 d + i: byte [s][t][h][i][d][b][y], nibble z.
    vc = vc.view(pairs, tiles, 2, 2, 2, 2, 2, 2, 4, 16).permute(0, 1, 2, 3, 5, 9, 8, 4, 6, 7)
    kc, vc = ((c[..., 0] | c[..., 1] << 4).reshape(pairs, tiles, 2048) for c in (kc, vc))
    # Keys' exponents [32 dims][a][i][s][b], values' [i][s][d], as e + 127.
    ke = ke.view(pairs, tiles, 2, 2, 2, 8, 2).permute(0, 1, 6, 3, 5, 2, 4).reshape(pairs, tiles, 128)
    ve = ve.view(pairs, tiles, 2, 4, 16).permute(0, 1, 4, 2, 3).reshape(pairs, tiles, 128)
    blocks = torch.cat((kc, vc, (ke + 127).to(torch.uint8), (ve + 127).to(torch.uint8)), dim=2)
    bounds = torch.stack((low, high), dim=2).to(torch.int8).view(torch.uint8)
    return torch.cat((blocks.flatten(), bounds.flatten(), scales.contiguous().view(torch.uint8).flatten()))


def _parts(cache, shape):
    """Blocks [P, T, 4352], bounds [P, T, 2, 64] and their scales [P, 64] of the cache's bytes."""
    pairs, tiles = shape[0] * shape[1], -(-shape[2] // 64)
    blocks, bounds, scales = cache.split((pairs * tiles * 4352, pairs * tiles * 128, pairs * 256))
    return (blocks.view(pairs, tiles, 4352), bounds.view(torch.int8).view(pairs, tiles, 2, 64),
            scales.view(torch.float32).view(pairs, 64))


def _decoded(cache, shape):
    """Keys and values [P, T * 64, 64] that the cache holds."""
    blocks = _parts(cache, shape)[0]
    pairs, tiles, _ = blocks.shape
    kc, vc, ke, ve = blocks.split((2048, 2048, 128, 128), dim=2)
    kc, vc = (torch.stack((c & 15, c >> 4), dim=-1) for c in (kc, vc))
    kc = kc.view(pairs, tiles, 2, 4, 2, 8, 2, 8, 2).permute(0, 1, 2, 4, 6, 5, 3, 7, 8).reshape(pairs, tiles * 64, 64)
    vc = vc.view(pairs, tiles, 2, 2, 2, 16, 4, 2, 2, 2).permute(0, 1, 2, 3, 7, 4, 8, 9, 6, 5)
    ke = ke.view(pairs, tiles, 2, 2, 8, 2, 2).permute(0, 1, 5, 3, 6, 4, 2).reshape(pairs, tiles * 64, 2)
    ve = ve.view(pairs, tiles, 16, 2, 4).permute(0, 1, 3, 4, 2).reshape(pairs, tiles * 2, 64)
    ke, ve = ke.int().sub_(127).repeat_interleave(32, dim=2), ve.int().sub_(127).repeat_interleave(32, dim=1)
    return _values(kc, ke), _values(vc.reshape(pairs, tiles * 64, 64), ve)


def _attended(state, rows):
    """Truth values [E, rows]: the rows that the estimator's queries attend to."""
    e, _, n = state["shape"]
    row = torch.arange(rows, device=state["q"].device)
    attended = (row < n).expand(e, rows)
    if state["lengths"] is not None:
        attended = attended & (row < state["lengths"][:, None])
    if state["keep"] is not None:
        bits = state["keep"][:, :, None] >> torch.arange(64, device=row.device) & 1
        attended = attended & bits.flatten(1).bool()
    return attended


def _softmax(scores, v, q):
    """Weighted values and log-sum-exp of scores (-inf: not attended), zero
    and -inf where nothing is."""
    largest = scores.amax(-1, keepdim=True)
    largest = largest.masked_fill(largest == -math.inf, 0.0)
    p = (scores - largest).exp()
    total = p.sum(-1, keepdim=True)
    out = (p.unsqueeze(-2) @ v).squeeze(-2) if v.dim() > scores.dim() else p @ v
    out = out / total.masked_fill(total == 0, 1.0)
    lse = (largest + total.log()).squeeze(-1)
    return out.view(q.shape).to(q.dtype), lse.view(q.shape[:3])


def _attend_plain(state):
    q, (e, h, _) = state["q"], state["shape"]
    k, v = _decoded(state["cache"], state["shape"])
    scores = q.float().flatten(0, 1) @ k.mT.contiguous() * SCALE
    attended = _attended(state, k.shape[1]).repeat_interleave(h, dim=0)
    return _softmax(scores.masked_fill(~attended[:, None], -math.inf), v, q)


def _select_plain(state):
    q, (e, h, n), count = state["q"], state["shape"], state["blocks"]
    _, bounds, scales = _parts(state["cache"], state["shape"])
    pairs, tiles = bounds.shape[:2]
    x = q.float().flatten(0, 1) * scales[:, None]
    part, power = torch.frexp(x.abs().amax(-1, keepdim=True))
    f = torch.where(part <= 127.0 / 128.0, power - 7, power - 6).clamp(min=-100)
    codes = (x * _pow2(-f)).round()
    low, high = bounds[:, :, 0].float(), bounds[:, :, 1].float()
    # Whole numbers below 2^24: exact in any order.
    scores = codes.clamp(min=0) @ high.mT.contiguous() + codes.clamp(max=0) @ low.mT.contiguous()
    some = _attended(state, tiles * 64).view(e, tiles, 64).any(-1).repeat_interleave(h, dim=0)[:, None]
    index = torch.arange(tiles, device=q.device)
    key = scores.long() * tiles + (tiles - 1 - index)
    key = key.masked_fill(~some, -(1 << 62))
    best = key.topk(min(count, tiles), dim=-1)
    picked = best.indices.masked_fill(best.values == -(1 << 62), tiles).sort(-1).values
    picked = torch.nn.functional.pad(picked, (0, count - picked.shape[-1]), value=tiles)
    return picked.masked_fill(picked == tiles, -1).int().view(e, h, q.shape[2], count)


def _choose_plain(state):
    q, (e, h, _) = state["q"], state["shape"]
    picked = _select_plain(state)
    k, v = _decoded(state["cache"], state["shape"])
    pairs, tiles = k.shape[0], k.shape[1] // 64
    at = picked.view(pairs, -1).long()
    pair = torch.arange(pairs, device=q.device)[:, None]
    some = _attended(state, tiles * 64).view(e, tiles, 64).repeat_interleave(h, dim=0)
    some = (some[pair, at.clamp(min=0)] & (at >= 0)[..., None]).view(pairs, q.shape[2], -1)
    k, v = (c.view(pairs, tiles, 4096)[pair, at.clamp(min=0)].view(pairs, q.shape[2], -1, 64) for c in (k, v))
    scores = (k @ q.float().flatten(0, 1).unsqueeze(-1)).squeeze(-1) * SCALE
    out, lse = _softmax(scores.masked_fill(~some, -math.inf), v, q)
    return picked, out, lse


def _store_plain(state):
    k, v, lengths, (e, h, n) = state["k"], state["v"], state["lengths"], state["shape"]
    kc, ke, vc, ve = _quantized(k, v, lengths)
    kv, vv = _values(kc, ke.repeat_interleave(32, dim=2)), _values(vc, ve.repeat_interleave(32, dim=1))
    low, high, scales = _bounds(kv, n, lengths, h)
    bounds = torch.stack((low * scales[:, None], high * scales[:, None]), dim=2)
    back = [x.view(e, h, -1, 64)[:, :, :n].to(k.dtype) for x in (kv, vv)]
    return back[0], back[1], bounds


# ---- the framework's calls ----

@functools.lru_cache(maxsize=None)
def _icl4():
    from ironicl_amd import hip, icl4
    return icl4, hip.Device(torch.cuda.current_device())


def _strides(x):
    return x.stride()[:3]


def _workspace(state):
    """Kept with the state, as a program keeps it with its context."""
    if "workspace" not in state:
        icl4, device = _icl4()
        size = icl4.workspace_bytes(device, state["shape"], state["q"].shape[2], state["blocks"])
        state["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return state["workspace"]


def _store_own(state):
    icl4, device = _icl4()
    k, v, lengths, shape = state["k"], state["v"], state["lengths"], state["shape"]
    stream = torch.cuda.current_stream().cuda_stream
    cache = torch.empty(icl4.cache_bytes(shape), dtype=torch.uint8, device="cuda")
    kind = {"element": "f16" if k.dtype == torch.float16 else "f32", "lengths": lengths, "stream": stream}
    icl4.encode(device, shape, k, v, cache, k_strides=_strides(k), v_strides=_strides(v), **kind)
    fresh = torch.empty if lengths is None else torch.zeros
    back = [fresh(k.shape, dtype=k.dtype, device="cuda") for _ in range(2)]
    bounds = torch.empty(shape[0] * shape[1], -(-shape[2] // 64), 2, 64, device="cuda")
    icl4.decode(device, shape, cache, back[0], back[1], bounds=bounds, **kind)
    return back[0], back[1], bounds


def _choose_own(state):
    icl4, device = _icl4()
    q, shape, count = state["q"], state["shape"], state["blocks"]
    work = _workspace(state)
    kind = {"element": "f16" if q.dtype == torch.float16 else "f32", "q_strides": _strides(q),
            "lengths": state["lengths"], "keep": state["keep"], "workspace": work, "workspace_bytes": work.numel(),
            "stream": torch.cuda.current_stream().cuda_stream}
    out = torch.empty_strided(q.shape, q.stride(), dtype=q.dtype, device="cuda")
    lse = torch.empty(q.shape[:3], device="cuda")
    picked = None
    if count:
        picked = torch.empty(q.shape[:3] + (count,), dtype=torch.int32, device="cuda")
        icl4.select(device, shape, state["cache"], q, q.shape[2], count, picked, **kind)
    icl4.attention(device, shape, state["cache"], q, q.shape[2], out, out_strides=_strides(out), scale=SCALE,
                   blocks=picked, n_blocks=count, lse=lse, **kind)
    return (picked, out, lse) if count else (out, lse)


def run(state):
    kind = state["kind"]
    if own:
        return _store_own(state) if kind == "store" else _choose_own(state)
    if kind == "store":
        return _store_plain(state)
    return _attend_plain(state) if kind == "attend" else _choose_plain(state)


# ---- the same in 64 bits, from the definitions ----

def _pow64(e):
    return (e + 1023 << 52).view(torch.float64)


def _held64(x, dim, lengths):
    """Values [E, H, N, 64] as the cache holds them, groups of 32 along `dim`
    (3: dims of one key, 2: rows of one dim), rows past the length zero."""
    x = x.double()
    e, h, n, d = x.shape
    if lengths is not None:
        x = x * (torch.arange(n, device=x.device) < lengths[:, None])[:, None, :, None]
    size = x.shape[dim]
    x = x.movedim(dim, -1)
    padded = torch.zeros(x.shape[:-1] + (-(-size // 32) * 32,), dtype=torch.float64, device=x.device)
    padded[..., :size] = x
    groups = padded.unflatten(-1, (-1, 32))
    top = groups.abs().amax(-1, keepdim=True)
    unit = torch.full_like(top, 2.0 ** -13)
    for power in range(-12, 14):
        unit = torch.where(top > 6.0 * 2.0 ** (power - 1), 2.0 ** power, unit)
    m = (groups.abs() / unit).clamp(max=6.0)
    step = torch.where(m < 2.0, 0.5, torch.where(m < 4.0, 1.0, 2.0))
    held = (m / step).round() * step * groups.sign() * unit
    return held.flatten(-2)[..., :size].movedim(-1, dim)


def _bounds64(k, lengths):
    """[E, H, T, 2, 64] whole numbers and the scales [E, H, 64] of held keys k."""
    e, h, n, _ = k.shape
    tiles = -(-n // 64)
    peak = k.abs().amax(2)
    unit = torch.full_like(peak, 2.0 ** -20)
    for power in range(-19, 12):
        unit = torch.where(peak > 127.0 * 2.0 ** (power - 1), 2.0 ** power, unit)
    out = torch.zeros(e, h, tiles, 2, 64, dtype=torch.float64, device=k.device)
    for i in range(e):
        rows = n if lengths is None else int(lengths[i])
        whole = rows // 64 * 64
        if whole:
            t = k[i, :, :whole].unflatten(1, (-1, 64))
            out[i, :, : whole // 64, 0], out[i, :, : whole // 64, 1] = t.amin(2), t.amax(2)
        if whole < rows:
            t = k[i, :, whole:rows]
            out[i, :, whole // 64, 0], out[i, :, whole // 64, 1] = t.amin(1), t.amax(1)
    out = out / unit[:, :, None, None]
    return torch.stack((out[..., 0, :].floor(), out[..., 1, :].ceil()), dim=3), unit


def _attend64(q, k, v, attended):
    """Output and log-sum-exp of q [Q, 64] over k, v [N, 64], attended [N] or [Q, N]."""
    out = torch.zeros(q.shape[0], 64, dtype=torch.float64, device=q.device)
    lse = torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
    step = max(1, int(2e8 / k.shape[0]))
    kt = k.t().contiguous()
    for r in range(0, q.shape[0], step):
        some = attended[r:r + step] if attended.dim() == 2 else attended[None]
        scores = (q[r:r + step] @ kt * SCALE).masked_fill(~some, -math.inf)
        lse[r:r + step] = scores.logsumexp(-1)
        out[r:r + step] = (scores - lse[r:r + step, None]).exp().nan_to_num(0.0) @ v
    return out, lse


def exact(case, seed):
    k, v, q, lengths, keep = _sources(case, seed)
    e, h, n, _ = k.shape
    k, v = _held64(k, 3, lengths), _held64(v, 2, lengths)
    if case["kind"] == "store":
        whole, unit = _bounds64(k, lengths)
        return k, v, (whole * unit[:, :, None, None]).flatten(0, 1)
    attended = torch.ones(e, n, dtype=torch.bool, device=k.device) if keep is None else keep
    if lengths is not None:
        attended = attended & (torch.arange(n, device=k.device) < lengths[:, None])
    q64 = q.double()
    outs, sums, picks = [], [], []
    tiles = -(-n // 64)
    if case["kind"] == "choose":
        whole, unit = _bounds64(k, lengths)
    for i in range(e):
        for j in range(h):
            some = attended[i]
            if case["kind"] == "choose":
                x = q64[i, j] * unit[i, j]
                top = x.abs().amax(-1, keepdim=True)
                f = torch.log2(top / 127.0).round().clamp(min=-100).long()  # within one of the smallest
                f = f + (top > 127.0 * _pow64(f)).long()
                f = (f - (top <= 127.0 * _pow64(f - 1)).long()).clamp(min=-100)
                codes = (x / _pow64(f)).round()
                low, high = whole[i, j, :, 0], whole[i, j, :, 1]
                scores = torch.zeros(q.shape[2], tiles, dtype=torch.float64, device=k.device)
                for d in range(64):
                    c = codes[:, d, None]
                    scores += torch.maximum(c * low[None, :, d], c * high[None, :, d])
                full = torch.zeros(tiles * 64, dtype=torch.bool, device=k.device)
                full[:n] = some
                scores[:, ~full.view(tiles, 64).any(-1)] = -math.inf
                order = scores.sort(dim=-1, descending=True, stable=True)
                index = order.indices.masked_fill(order.values == -math.inf, tiles)[:, : case["blocks"]]
                index = index.sort(-1).values
                pick = torch.full((q.shape[2], case["blocks"]), -1, dtype=torch.int32, device=k.device)
                pick[:, : index.shape[1]] = index.masked_fill(index == tiles, -1)
                picks.append(pick)
                listed_blocks = torch.zeros(q.shape[2], tiles + 1, dtype=torch.bool, device=k.device)
                listed_blocks.scatter_(1, index, True)
                of = torch.arange(n, device=k.device) // 64
                some = listed_blocks[:, of] & some
            o, s = _attend64(q64[i, j], k[i, j], v[i, j], some)
            outs.append(o), sums.append(s)
    out, lse = (torch.stack(x).unflatten(0, (e, h)) for x in (outs, sums))
    return (torch.stack(picks).unflatten(0, (e, h)), out, lse) if case["kind"] == "choose" else (out, lse)
