"""What is measured of the calls for training: attention that keeps what its
backward pass needs, that backward pass, and dropout.

Three kinds of case, over the public entry points:

  attend    irx_train_attention: D(softmax(q k^T / 8)) v and the log-sum-exp
            over each estimator's rows, D the weights' dropout.
  gradient  irx_train_attention_backward: the gradients of q, k and v from that
            of the output, the probabilities computed anew.
  drop      irx_train_dropout: residual + D(x), or D(x) alone, which is its own
            backward pass.

Which numbers are dropped follows from the seed: Philox4x32 with seven rounds
(Salmon, Moraes, Dror and Shaw, SC 2011), laid out as the library's header
states. Sizes are those of the benchmark's contexts (1,024 and 50,000 training
rows, 512 wide) and of odd tables between.

torch is imported before the backend, so that both use one HIP runtime.
"""

import functools
import math

import torch

own = False

SCALE = 0.125  # 1 / sqrt(64)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One row against the benchmark's context: keys and values are read once.
        {"name": "attend_row", "kind": "attend", "estimators": 1, "kv_heads": 8, "queries": 1, "rows": 50000,
         "element": "f32", "layout": "heads", "ragged": False, "masked": False, "dropped": 0},
        # A few dozen rows over two small tables: latency.
        {"name": "attend_small", "kind": "attend", "estimators": 2, "kv_heads": 8, "queries": 33, "rows": 1024,
         "element": "f32", "layout": "heads", "ragged": False, "masked": False, "dropped": 6554},
        # A 512-row pass over the benchmark's context.
        {"name": "attend_pass", "kind": "attend", "estimators": 1, "kv_heads": 8, "queries": 512, "rows": 50000,
         "element": "f32", "layout": "heads", "ragged": False, "masked": False, "dropped": 0},
        # A table of 10,007 rows attending to itself, as token rows of a mixed-precision step with dropout.
        {"name": "attend_self", "kind": "attend", "estimators": 1, "kv_heads": 8, "queries": 10007, "rows": 10007,
         "element": "bf16", "layout": "tokens", "ragged": False, "masked": False, "dropped": 6554},
        # The gradients of the small tables' step.
        {"name": "gradient_small", "kind": "gradient", "estimators": 2, "kv_heads": 8, "queries": 33, "rows": 1024,
         "element": "f32", "layout": "heads", "ragged": False, "masked": False, "dropped": 6554},
        # Four tables of 1,024 rows in a batch, FP32 with dropout: an ordinary step.
        {"name": "gradient_batch", "kind": "gradient", "estimators": 4, "kv_heads": 8, "queries": 1024, "rows": 1024,
         "element": "f32", "layout": "tokens", "ragged": False, "masked": False, "dropped": 6554},
        # The context's own gradients from 512 rows: tuning 50,000 rows' keys and values.
        {"name": "gradient_pass", "kind": "gradient", "estimators": 1, "kv_heads": 8, "queries": 512, "rows": 50000,
         "element": "f32", "layout": "heads", "ragged": False, "masked": False, "dropped": 0},
        # Two padded tables of different lengths with rows held out, four heads to a key head, FP16 token rows.
        {"name": "gradient_masked", "kind": "gradient", "estimators": 2, "kv_heads": 2, "queries": 777, "rows": 12345,
         "element": "f16", "layout": "tokens", "ragged": True, "masked": True, "dropped": 6554},
        # The table of 10,007 rows, its gradients.
        {"name": "gradient_self", "kind": "gradient", "estimators": 1, "kv_heads": 8, "queries": 10007, "rows": 10007,
         "element": "bf16", "layout": "tokens", "ragged": False, "masked": False, "dropped": 0},
        # A small table's block output onto its residual: latency.
        {"name": "drop_small", "kind": "drop", "rows": 1024, "width": 512, "element": "f32", "residual": True,
         "dropped": 6554},
        # The benchmark's 50,000 rows in BF16.
        {"name": "drop_context", "kind": "drop", "rows": 50000, "width": 512, "element": "bf16", "residual": True,
         "dropped": 6554},
        # The feed-forward half's 1,024 columns over an ensemble of four, without a residual: a backward pass.
        {"name": "drop_ensemble", "kind": "drop", "rows": 200000, "width": 1024, "element": "f32", "residual": False,
         "dropped": 19661},
    ]


# ---- draws ----

def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed kinds: sizes uniform in their logarithm, no dearer
    than the dearest listed one of its kind. Gradients are of two dozen rows at
    least: where a query attends to one alone, its weight is 1 whatever the
    scores are, and what any form returns for q and k is rounding."""
    while True:
        kind = rng.choice(("attend", "attend", "gradient", "gradient", "drop"))
        element = rng.choice(("f32", "f16", "bf16"))
        dropped = rng.choice((0, 0, 655, 6554, 19661, 32768))
        if kind == "drop":
            case = {"kind": kind, "rows": _log(rng, 1, 200000), "width": _log(rng, 1, 1024), "element": element,
                    "residual": rng.random() < 0.5, "dropped": dropped}
        else:
            case = {"kind": kind, "estimators": rng.randint(1, 4), "kv_heads": rng.choice((8, 8, 2, 1)),
                    "queries": _log(rng, 1, 10007), "rows": _log(rng, 24 if kind == "gradient" else 1, 200000),
                    "element": element, "layout": rng.choice(("heads", "tokens")),
                    "ragged": rng.random() < 0.4, "masked": rng.random() < 0.4, "dropped": dropped}
            if case["estimators"] * case["rows"] > 400000:
                continue
        if _held(case) <= max(_held(c) for c in listed() if c["kind"] == kind):
            return case


def _held(case):
    """Numbers that the plain form holds at once."""
    if case["kind"] == "drop":
        return case["rows"] * case["width"]
    return 8 * case["estimators"] * (case["queries"] * case["rows"] + 64 * (case["queries"] + case["rows"]))


# ---- work ----

def work(case):
    size = 4 if case["element"] == "f32" else 2
    if case["kind"] == "drop":
        return {"bytes": float(case["rows"] * case["width"] * size * (3 if case["residual"] else 2)), "flops": 0.0}
    e, n, rows = case["estimators"], case["rows"], case["queries"]
    q, kv = 8 * e * rows * 64 * size, case["kv_heads"] * e * n * 64 * size
    masks = e * -(-n // 64) * 8 if case["masked"] else 0
    if case["kind"] == "attend":
        return {"bytes": float(2 * q + 2 * kv + 8 * e * rows * 4 + masks), "flops": 4.0 * 64 * 8 * e * rows * n}
    return {"bytes": float(4 * q + 4 * kv + 8 * e * rows * 8 + masks), "flops": 10.0 * 64 * 8 * e * rows * n}


# ---- inputs ----

def _rows(case, g, heads, rows):
    """[E, heads, rows, 64] standard normal, as one head after another or as views of token rows."""
    e = case["estimators"]
    if case["layout"] == "tokens":
        return torch.randn(e, rows, heads, 64, generator=g, device="cuda").transpose(1, 2)
    return torch.randn(e, heads, rows, 64, generator=g, device="cuda")


def _sources(case, seed):
    """q, k, v, the output's gradient, lengths of queries and rows (or None),
    kept rows (or None) and the dropout's seed. Channels differ in size, as
    learned ones do."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    e, n, rows, kv = case["estimators"], case["rows"], case["queries"], case["kv_heads"]
    kind = TYPES[case["element"]]
    gain = torch.exp(0.4 * torch.randn(e, kv, 1, 64, generator=g, device="cuda"))
    k = _rows(case, g, kv, n).mul_(gain).to(kind)
    v = _rows(case, g, kv, n).to(kind)
    q = _rows(case, g, 8, rows).mul_(1.3).to(kind)
    # The gradient of a loss's mean over the rows, scaled as half-precision steps scale it.
    dout = _rows(case, g, 8, rows).mul_(2.0 ** -6).to(kind) if case["kind"] == "gradient" else None
    lengths = query_lengths = keep = None
    if case["ragged"]:
        lengths = torch.randint(n // 2, n + 1, (e,), generator=g, device="cuda", dtype=torch.int32)
        query_lengths = torch.randint(rows // 2, rows + 1, (e,), generator=g, device="cuda", dtype=torch.int32)
        if e > 2:
            lengths[-1] = 0  # an estimator without rows
    if case["masked"]:
        keep = torch.rand(e, n, generator=g, device="cuda") < 0.8
        keep &= torch.rand(e, -(-n // 200), generator=g, device="cuda")[:, torch.arange(n, device="cuda") // 200] < 0.9
    number = torch.randint(-(1 << 62), 1 << 62, (1,), generator=g, device="cuda")
    return q, k, v, dout, query_lengths, lengths, keep, number


def _drop_sources(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, shape = TYPES[case["element"]], (case["rows"], case["width"])
    pitch = -(-shape[1] // 8) * 8  # rows start at whole 16 bytes
    x, residual = (torch.randn(shape[0], pitch, generator=g, device="cuda").to(kind)[:, : shape[1]] for _ in range(2))
    number = torch.randint(-(1 << 62), 1 << 62, (1,), generator=g, device="cuda")
    return x, residual if case["residual"] else None, number


def _bits(keep):
    """[E, N] truth values as 64-bit words, row r at bit r % 64 of word r / 64."""
    e, n = keep.shape
    padded = torch.zeros(e, -(-n // 64) * 64, dtype=torch.int64, device=keep.device)
    padded[:, :n] = keep
    return (padded.view(e, -1, 64) << torch.arange(64, device=keep.device)).sum(-1)


def prepare(case, seed):
    """Inputs and, for gradients, what the forward pass left: its output and
    its statistics. Rows past the lengths are not written: they start as zeros."""
    if case["kind"] == "drop":
        x, residual, number = _drop_sources(case, seed)
        state = {"kind": "drop", "x": x, "residual": residual, "seed": number, "dropped": case["dropped"],
                 "out": torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")}
        torch.cuda.synchronize()
        return state
    q, k, v, dout, query_lengths, lengths, keep, number = _sources(case, seed)
    state = {"kind": case["kind"], "q": q, "k": k, "v": v, "dout": dout, "query_lengths": query_lengths,
             "lengths": lengths, "keep": None if keep is None else _bits(keep), "seed": number,
             "dropped": case["dropped"], "element": case["element"]}
    zeros = lambda x: torch.zeros_like(x, memory_format=torch.preserve_format)  # noqa: E731
    if case["kind"] == "gradient":
        state["out"], _, state["stats"] = _attend_plain(state)
        state["out"] = zeros(q).copy_(state["out"])
        state["gradients"] = [zeros(x) for x in (q, k, v)]
    else:
        state["out"], state["lse"] = zeros(q), torch.zeros(q.shape[:3], device="cuda")
        state["stats"] = torch.zeros(q.shape[:3] + (2,), device="cuda")
    torch.cuda.synchronize()
    return state


# ---- the plain forms ----

def _philox(counter, seed):
    """Four words (whole numbers below 2^32) of counters (four of them, alike) and the 64-bit seed."""
    low = 0xFFFFFFFF
    a, b, c, d = counter
    x, y = seed & low, (seed >> 32) & low
    for _ in range(7):
        p, r = a * 0xD2511F53, c * 0xCD9E8D57  # modulo 2^64
        a, b, c, d = ((r >> 32) & low) ^ b ^ x, r & low, ((p >> 32) & low) ^ d ^ y, p & low
        x, y = (x + 0x9E3779B9) & low, (y + 0xBB67AE85) & low
    return a, b, c, d


def _values(counter, seed):
    """Eight 16-bit numbers a call, in a last axis: the words' low halves first."""
    words = torch.stack(_philox(counter, seed), dim=-1)
    return torch.stack((words & 0xFFFF, words >> 16), dim=-1).flatten(-2)


def _kept_weights(state, n):
    """Truth values [E, H, Q, N]: the weights that are not dropped."""
    e, h, rows = state["q"].shape[:3]
    at = lambda count, axis: torch.arange(count, device="cuda").view([-1 if i == axis else 1 for i in range(3)])  # noqa: E731
    site = torch.zeros((), dtype=torch.int64, device="cuda")
    cells = -(-n // 16) * 2
    counter = (at(cells, 2), at(rows, 1), at(e * h, 0), site)
    kept = _values(torch.broadcast_tensors(*counter), state["seed"]) >= state["dropped"]
    # Cell 2 c + i, value 4 b + j: key 16 c + 8 b + 4 i + j.
    kept = kept.view(e, h, rows, cells // 2, 2, 2, 4).transpose(4, 5)
    return kept.reshape(e, h, rows, -1)[..., :n]


def _attended(state, n):
    """Truth values [E, 1, 1, N]: the rows that the estimator's queries attend to."""
    row = torch.arange(n, device="cuda")
    attended = (row >= 0).expand(state["q"].shape[0], n)
    if state["lengths"] is not None:
        attended = attended & (row < state["lengths"][:, None])
    if state["keep"] is not None:
        bits = state["keep"][:, :, None] >> torch.arange(64, device="cuda") & 1
        attended = attended & bits.flatten(1)[:, :n].bool()
    return attended[:, None, None]


def _inside(state):
    """Truth values [E, 1, Q, 1]: the rows that are queries."""
    row = torch.arange(state["q"].shape[2], device="cuda")
    lengths = state["query_lengths"]
    inside = (row >= 0)[None] if lengths is None else row < lengths[:, None]
    return inside[:, None, :, None]


def _shared(x, heads, attended):
    """Keys or values in FP32, one to each of `heads`, zero where none attends."""
    x = x.float().masked_fill(~attended.transpose(2, 3), 0.0)
    return x.repeat_interleave(heads // x.shape[1], dim=1).contiguous()


def _scores(state, k, attended):
    """log2(e) q k^T / 8, -inf where not attended."""
    x = (state["q"].float().contiguous() @ k.mT.contiguous()) * (SCALE * math.log2(math.e))
    return x.masked_fill_(~attended, -math.inf)


def _attend_plain(state):
    q = state["q"]
    attended = _attended(state, state["k"].shape[2])
    k, v = (_shared(state[x], q.shape[1], attended) for x in "kv")
    x = _scores(state, k, attended)
    top = x.amax(-1, keepdim=True).ceil()
    top = top.masked_fill(top == -math.inf, 0.0)
    p = (x - top).exp2()
    total = p.sum(-1, keepdim=True)
    if state["dropped"]:
        p = p * _kept_weights(state, p.shape[-1]) * (65536.0 / (65536 - state["dropped"]))
    out = (p @ v) / total.masked_fill(total == 0, 1.0)
    lse = ((top + total.log2()) * math.log(2.0)).squeeze(-1)
    inside = _inside(state)
    stats = torch.cat((top, total), dim=-1).masked_fill(~inside, 0.0)
    return out.masked_fill(~inside, 0.0).to(q.dtype), lse.masked_fill(~inside[..., 0], 0.0), stats


def _gradient_plain(state):
    q, inside, heads = state["q"], _inside(state), state["q"].shape[1]
    attended = _attended(state, state["k"].shape[2])
    k, v = (_shared(state[x], heads, attended) for x in "kv")
    top, total = state["stats"].split(1, dim=-1)
    p = (_scores(state, k, attended) - top).exp2() / total.masked_fill(total == 0, 1.0)
    p = p.masked_fill_(~inside, 0.0)
    dout = state["dout"].float().masked_fill(~inside, 0.0).contiguous()
    delta = (dout * state["out"].float().masked_fill(~inside, 0.0)).sum(-1, keepdim=True)
    dp = dout @ v.mT.contiguous()
    dropped = p
    if state["dropped"]:
        kept = _kept_weights(state, p.shape[-1]) * (65536.0 / (65536 - state["dropped"]))
        dropped, dp = p * kept, dp * kept
    dv = dropped.mT.contiguous() @ dout
    ds = p * (dp - delta)
    dq = ds @ k * SCALE
    dk = ds.mT.contiguous() @ q.float().masked_fill(~inside, 0.0).contiguous() * SCALE
    groups = state["k"].shape[1]
    dk, dv = (x.unflatten(1, (groups, heads // groups)).sum(2) for x in (dk, dv))
    return dq.to(q.dtype), dk.to(q.dtype), dv.to(q.dtype)


def _drop_plain(state):
    x, residual = state["x"], state["residual"]
    out = x.float()
    if state["dropped"]:
        rows, width = x.shape
        counter = (torch.arange(-(-width // 8), device="cuda"), torch.arange(rows, device="cuda")[:, None],
                   torch.full((), 0xFFFFFFFF, device="cuda"), torch.zeros((), dtype=torch.int64, device="cuda"))
        kept = _values(torch.broadcast_tensors(*counter), state["seed"]).flatten(1)[:, :width] >= state["dropped"]
        out = out * kept * (65536.0 / (65536 - state["dropped"]))
    if residual is not None:
        out = out + residual.float()
    return out.to(x.dtype)


# ---- the framework's calls ----

@functools.lru_cache(maxsize=None)
def _training():
    from ironicl_amd import hip, training
    return training, hip.Device(torch.cuda.current_device())


def _strides(x):
    return x.stride()[:3]


def _own(state):
    training, device = _training()
    stream = torch.cuda.current_stream().cuda_stream
    drop = {"seed": state["seed"], "dropped": state["dropped"], "stream": stream}
    if state["kind"] == "drop":
        x, out, residual = state["x"], state["out"], state["residual"]
        kind = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[x.dtype]
        training.dropout(device, x.shape[0], x.shape[1], x, out, element=kind, residual=residual, x_stride=x.stride(0),
                         residual_stride=None if residual is None else residual.stride(0), out_stride=out.stride(0),
                         **drop)
        return out
    q, k, v, out = state["q"], state["k"], state["v"], state["out"]
    backward = state["kind"] == "gradient"
    shape = (q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2])
    if "workspace" not in state:  # kept with the state, as a program keeps it with its layer
        size = training.workspace_bytes(device, shape, element=state["element"], backward=backward)
        state["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    work = state["workspace"]
    kind = {"element": state["element"], "scale": SCALE, "q_strides": _strides(q), "k_strides": _strides(k),
            "v_strides": _strides(v), "out_strides": _strides(out), "query_lengths": state["query_lengths"],
            "lengths": state["lengths"], "keep": state["keep"], "workspace": work, "workspace_bytes": work.numel()}
    if not backward:
        training.attention(device, shape, q, k, v, out, stats=state["stats"], lse=state["lse"], **kind, **drop)
        return out, state["lse"]
    dq, dk, dv = state["gradients"]
    training.attention_backward(device, shape, q, k, v, out, state["stats"], state["dout"], dq=dq, dk=dk, dv=dv,
                                dout_strides=_strides(state["dout"]), dq_strides=_strides(dq),
                                dk_strides=_strides(dk), dv_strides=_strides(dv), **kind, **drop)
    return dq, dk, dv


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "drop":
        return _drop_plain(state)
    return _gradient_plain(state) if state["kind"] == "gradient" else _attend_plain(state)[:2]


# ---- the same in 64 bits, from the definitions ----

def _random16(c0, c1, c2, seed, index):
    """The 16-bit number `index` (0 to 7) of the call with counters c0, c1, c2 and 0, broadcast."""
    def high_low(x, m):  # of x * m in halves of 16 bits, nothing past 2^48
        x0, x1, m0, m1 = x % 65536, x // 65536, m % 65536, m // 65536
        middle = x0 * m0 // 65536 + (x1 * m0) % 65536 + (x0 * m1) % 65536
        top = x1 * m1 + x1 * m0 // 65536 + x0 * m1 // 65536 + middle // 65536
        return top, (middle % 65536) * 65536 + (x0 * m0) % 65536

    seed %= 1 << 64
    keys = [seed % (1 << 32), seed >> 32]
    w = list(torch.broadcast_tensors(c0, c1, c2, torch.zeros_like(c0)))
    for _ in range(7):
        h0, l0 = high_low(w[0], 0xD2511F53)
        h1, l1 = high_low(w[2], 0xCD9E8D57)
        w = [h1 ^ w[1] ^ keys[0], l1, h0 ^ w[3] ^ keys[1], l0]
        keys = [(keys[0] + 0x9E3779B9) % (1 << 32), (keys[1] + 0xBB67AE85) % (1 << 32)]
    word = torch.where(index < 4, torch.where(index < 2, w[0], w[1]), torch.where(index < 6, w[2], w[3]))
    return torch.where(index % 2 == 0, word % 65536, word // 65536)


def _kept64(seed, dropped, pair, first, count, n):
    """1 / (1 - p) or 0 for the weights of queries `first` .. first + count - 1 and n rows of one (estimator, head)."""
    if not dropped:
        return 1.0
    groups = torch.arange(-(-n // 4), device="cuda")[None, :]  # of four rows: half a call's values
    query = first + torch.arange(count, device="cuda")[:, None]
    kept = []
    for j in range(4):
        number = _random16(groups // 4 * 2 + groups % 2, query, torch.full_like(groups, pair), seed,
                           groups % 4 // 2 * 4 + j)
        kept.append(number >= dropped)
    return torch.stack(kept, dim=-1).flatten(1)[:, :n].double() / (1.0 - dropped / 65536.0)


def exact(case, seed):
    if case["kind"] == "drop":
        x, residual, number = _drop_sources(case, seed)
        out = x.double()
        if case["dropped"]:
            column = torch.arange(case["width"], device="cuda")[None, :]
            row = torch.arange(case["rows"], device="cuda")
            step = max(1, int(3e7 / case["width"]))
            for r in range(0, case["rows"], step):
                number16 = _random16(column // 8, row[r:r + step, None], torch.full_like(column, 0xFFFFFFFF),
                                     int(number), column % 8)
                out[r:r + step] *= (number16 >= case["dropped"]).double() / (1.0 - case["dropped"] / 65536.0)
        return out if residual is None else out + residual.double()
    q, k, v, dout, query_lengths, lengths, keep, number = _sources(case, seed)
    e, h, rows, _ = q.shape
    n, kv = k.shape[2], k.shape[1]
    number = int(number)
    out, dq = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    lse = torch.zeros(q.shape[:3], dtype=torch.float64, device="cuda")
    dk, dv = (torch.zeros(k.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    step = max(1, int(1e8 / n))
    for i in range(e):
        count = n if lengths is None else int(lengths[i])
        queries = rows if query_lengths is None else int(query_lengths[i])
        some = torch.arange(count, device="cuda")
        if keep is not None:
            some = some[keep[i, :count]]
        for j in range(h):
            kk, vv = k[i, j // (h // kv), some].double(), v[i, j // (h // kv), some].double()
            for first in range(0, queries, step):
                at = slice(first, min(queries, first + step))
                if not len(some):
                    lse[i, j, at] = -math.inf
                    continue
                qq = q[i, j, at].double()
                scores = qq @ kk.t() * SCALE
                lse[i, j, at] = scores.logsumexp(-1)
                p = (scores - lse[i, j, at, None]).exp()
                z = _kept64(number, case["dropped"], i * h + j, first, len(qq), n)
                z = z if isinstance(z, float) else z[:, some]
                o = (p * z) @ vv
                out[i, j, at] = o
                if dout is None:
                    continue
                g = dout[i, j, at].double()
                dv[i, j // (h // kv)].index_add_(0, some, (p * z).t() @ g)
                ds = p * (g @ vv.t() * z - (g * o).sum(-1, keepdim=True))
                dq[i, j, at] = ds @ kk * SCALE
                dk[i, j // (h // kv)].index_add_(0, some, ds.t() @ qq * SCALE)
    return (out, lse) if dout is None else (dq, dk, dv)
