"""Cases that measure the table operators and the dropout: embedding lookup
with scaling (and dropout in the same pass), its gradient by sorted tokens,
the gradient handed straight to Adam, and dropout from a counter-based
generator.

`own = False` computes them in plain torch operations, `own = True` calls the
framework's modules `embedding` and `dropout`.
"""

import functools
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
INDEX = {"i32": torch.int32, "i64": torch.int64}
RATE, STEP = 0.0025, 200  # learning rate and 1-based step of the Adam cases
BIAS1, BIAS2_SQRT = 1.0 - 0.9 ** STEP, math.sqrt(1.0 - 0.999 ** STEP)
EPS = 1e-15
LONG = 1 << 17  # from this many tokens on, a row's sum is long enough to need 64 bits


def _lookup(name, tokens, rows, width, dtype, index, **more):
    return {"name": name, "op": "lookup", "tokens": tokens, "rows": rows, "width": width,
            "dtype": dtype, "index": index, "scale": 1.0, "p": 0.0, "padding": False,
            "gap": 0, **more}


def _dropout(name, tokens, width, dtype, **more):
    return {"name": name, "op": "dropout", "tokens": tokens, "width": width, "dtype": dtype,
            "p": 0.1, "rows_form": False, "backward": False, "gap": 0, **more}


def listed():
    return [
        # One token of a language-sized table: the latency of the smallest call.
        _lookup("lookup, one token", 1, 65536, 2048, "bf16", "i64", scale=math.sqrt(2048.0)),
        # 1.1M Gaussians taking their 48 SH coefficients from a codebook.
        _lookup("lookup, codebook colours", 1_100_000, 4096, 48, "f32", "i32"),
        # A batch of token embeddings, scaled by the root of the width.
        _lookup("lookup, token batch", 16384, 131072, 2048, "bf16", "i64",
                scale=math.sqrt(2048.0)),
        # Odd sizes, padded tokens and dropout in the same pass.
        _lookup("lookup, odd with dropout", 100_003, 5003, 77, "f16", "i64", p=0.1,
                padding=True, scale=0.5),
        # The codebook's gradient: few rows, long sums, a few rows far more used than the rest.
        {**_lookup("gradient, codebook colours", 1_100_000, 4096, 48, "f32", "i32"),
         "op": "gradient"},
        # A large table of which a batch names a small part; the rest is zeros.
        {**_lookup("gradient, token batch", 16384, 131072, 2048, "bf16", "i64",
                   scale=math.sqrt(2048.0)), "op": "gradient"},
        # A small odd one: latency.
        {**_lookup("gradient, small", 37, 1000, 45, "f32", "i64", p=0.25, padding=True),
         "op": "gradient"},
        # The codebook's training step; assignments stay the same over the steps.
        {**_lookup("adam, codebook colours", 1_100_000, 8192, 48, "f32", "i32"),
         "op": "adam", "kept": True},
        # A token table's training step, bf16 gradients through the dropout.
        {**_lookup("adam, token batch", 8192, 32768, 1024, "bf16", "i64", p=0.1, scale=32.0),
         "op": "adam", "kept": False},
        # The opacities of 6M Gaussians.
        _dropout("dropout, opacities", 6_000_000, 1, "f32"),
        # Hidden states, forward and backward.
        _dropout("dropout, states", 16384, 4096, "bf16", backward=True),
        # Whole rows dropped, few and odd.
        _dropout("dropout, rows", 257, 33, "f16", rows_form=True, backward=True, p=0.5),
    ]


def _between(rng, low, high):
    """A whole number in [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["lookup", "gradient", "adam", "dropout"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    p = rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.9), 3)])
    gap = rng.choice([0, 0, 0, 5, 16])
    if op == "dropout":
        width = rng.choice([1, 3, 48, _between(rng, 1, 8192)])
        tokens = _between(rng, 1, max(1, min(6_000_000, 48_000_000 // (width + gap))))
        rows_form = rng.random() < 0.3
        return {"op": op, "tokens": tokens, "width": width, "dtype": dtype,
                "p": p or 0.1, "rows_form": rows_form, "backward": rng.random() < 0.5,
                "gap": gap if width > 1 else 0}
    width = rng.choice([3, 16, 48, _between(rng, 1, 4096)])
    rows = _between(rng, 1, min(131072, 100_000_000 // width))
    tokens = _between(rng, 1, max(1, min(1_100_000, 50_000_000 // (width + gap))))
    case = {"op": op, "tokens": tokens, "rows": rows, "width": width, "dtype": dtype,
            "index": rng.choice(["i32", "i64"]), "scale": rng.choice([1.0, 0.5, math.sqrt(width)]),
            "p": p, "padding": rng.random() < 0.3, "gap": gap}
    if op == "adam":
        case["rows"] = min(rows, max(1, 20_000_000 // width))
        case["kept"] = rng.random() < 0.5
    return case


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(rows, width, std, gap=0, kind=dtype):
        whole = torch.empty(rows, width + gap, dtype=kind, device="cuda")
        whole.normal_(0.0, std, generator=g)
        return whole[:, :width] if gap else whole

    n, d = case["tokens"], case["width"]
    s = {"case": case, "seed": int(torch.randint(0, 2 ** 62, (1,), generator=g, device="cuda")),
         "offset": int(torch.randint(0, 2 ** 40, (1,), generator=g, device="cuda"))}
    if case["op"] == "dropout":
        # Opacities lie in (0, 1); states around zero.
        s["x"] = normal(n, d, 1.0, case["gap"]) if d > 1 else torch.rand(
            n, 1, generator=g, device="cuda").to(dtype)
        if case["backward"]:
            s["grad"] = normal(n, d, 1.0)
        return s
    k = case["rows"]
    # A row's use falls with its rank; ranks are spread over the table.
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(k + 1.0)).to(torch.int64) - 1).clamp_(0, k - 1)
    place = torch.randperm(k, generator=g, device="cuda")
    index = place[rank]
    s["padding"] = None
    if case["padding"]:
        s["padding"] = -1
        index = torch.where(torch.rand(n, generator=g, device="cuda") < 0.1,
                            torch.full_like(index, -1), index)
    s["index"] = index.to(INDEX[case["index"]])
    if case["op"] == "lookup":
        s["table"] = normal(k, d, 0.05, case["gap"])
    else:
        s["grad"] = normal(n, d, 1e-3, case["gap"])
    if case["op"] == "adam":
        s["table"] = normal(k, d, 0.05, kind=torch.float32)
        s["first"] = normal(k, d, 1e-3, kind=torch.float32)
        s["second"] = torch.empty(k, d, device="cuda").uniform_(1e-6, 4e-6, generator=g)
    return s


def _modules():
    """The framework's modules (flat ones, in its package directory)."""
    package = str(Path(__file__).resolve().parents[1] / "clad-3dgs_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import dropout
    import embedding
    return embedding, dropout


def prepare(case, seed):
    s = _inputs(case, seed)
    s["order"] = None
    if own:
        s["embedding"], s["dropout"] = _modules()
        if case.get("kept"):
            # Assignments that stay the same over a training's steps: a
            # program sorts them once.
            s["order"] = s["embedding"].token_order(s["index"], case["rows"],
                                                    padding_index=s["padding"])
    if case.get("backward"):
        s["x"].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# Plain forms.

LOW = 0xFFFFFFFF


def _round(state, number):
    """One round of Philox4x32 on words held in int64 (products wrap, which
    leaves their 64 bits right)."""
    c0, c1, c2, c3, k0, k1 = state
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
    key0 = (k0 + number * 0x9E3779B9) & LOW
    key1 = (k1 + number * 0xBB67AE85) & LOW
    return (((b >> 32) & LOW) ^ c1 ^ key0, b & LOW, ((a >> 32) & LOW) ^ c3 ^ key1, a & LOW, k0, k1)


def _keep(count, p, seed, offset):
    """Which of `count` elements stay (bool)."""
    block = torch.arange((count + 3) // 4, device="cuda")
    state = (block & LOW, block >> 32, torch.full_like(block, offset & LOW),
             torch.full_like(block, offset >> 32), seed & LOW, seed >> 32)
    words = torch.stack(functools.reduce(_round, range(10), state)[:4], dim=1)
    return words.reshape(-1)[:count] >= int(p * 2.0 ** 32)


def _plain_dropout(s):
    case, x = s["case"], s["x"].detach()
    count = case["tokens"] if case["rows_form"] else x.numel()
    keep = _keep(count, case["p"], s["seed"], s["offset"])
    keep = keep.view(-1, 1) if case["rows_form"] else keep.view(x.shape)
    factor = 1.0 / (1.0 - case["p"])
    drop = lambda v: torch.where(keep, v.float() * factor, 0.0).to(v.dtype)
    return {"y": drop(x), "dx": drop(s["grad"])} if case["backward"] else drop(x)


def _factor(case):
    return case["scale"] / (1.0 - case["p"])


def _plain_lookup(s):
    case, table = s["case"], s["table"]
    index = s["index"].long()
    real = index >= 0
    y = table[index.clamp(min=0)].float() * _factor(case)
    if case["padding"]:
        y = torch.where(real.view(-1, 1), y, 0.0)
    if case["p"] > 0:
        y = torch.where(_keep(y.numel(), case["p"], s["seed"], s["offset"]).view(y.shape), y, 0.0)
    return y.to(table.dtype)


def _plain_sums(s):
    """The table's gradient in the precision it is summed in."""
    case, grad = s["case"], s["grad"]
    kind = torch.float64 if case["tokens"] >= LONG else torch.float32
    terms = grad.to(kind)
    if case["p"] > 0:
        keep = _keep(grad.shape[0] * grad.shape[1], case["p"], s["seed"], s["offset"])
        terms = torch.where(keep.view(grad.shape), terms, 0.0)
    index = s["index"].long()
    sums = torch.zeros(case["rows"] + 1, case["width"], dtype=kind, device="cuda")
    # Padded tokens add into a row behind the table.
    sums.index_add_(0, torch.where(index < 0, case["rows"], index), terms)
    return sums[:-1] * _factor(case)


def _plain_adam(s):
    g = _plain_sums(s).float()
    table, first, second = s["table"], s["first"], s["second"]
    first.mul_(0.9).add_(g * 0.1)
    second.mul_(0.999).add_(0.001 * g * g)
    table.sub_((RATE / BIAS1) * first / (second.sqrt() / BIAS2_SQRT + EPS))
    return {"table": table, "first": first, "second": second}


# ---------------------------------------------------------------------------

def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        if op == "dropout":
            return _plain_dropout(s)
        if op == "lookup":
            return _plain_lookup(s)
        if op == "gradient":
            return _plain_sums(s).to(s["grad"].dtype)
        return _plain_adam(s)
    if op == "dropout":
        y = s["dropout"].dropout(s["x"], case["p"], s["seed"], s["offset"],
                                 rows=case["rows_form"])
        if not case["backward"]:
            return y
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["grad"])[0]}
    how = dict(scale=case["scale"], padding_index=s["padding"], p=case["p"], seed=s["seed"],
               offset=s["offset"])
    if op == "lookup":
        return s["embedding"].lookup(s["table"], s["index"], **how)
    if op == "gradient":
        return s["embedding"].lookup_gradient(s["grad"], s["index"], case["rows"], **how)
    s["embedding"].consume_torch_adam(s["table"], s["first"], s["second"], s["grad"],
                                      s["index"], rate=RATE, bias1=BIAS1,
                                      bias2_sqrt=BIAS2_SQRT, order=s["order"], **how)
    return {"table": s["table"], "first": s["first"], "second": s["second"]}


def work(case):
    n, d, es = case["tokens"], case["width"], SIZES[case["dtype"]]
    # Philox: 10 rounds of two products and four exclusive-ors for four elements.
    mask = 15.0 if case["p"] > 0 else 0.0
    if case["op"] == "dropout":
        passes = 2 if case["backward"] else 1
        drawn = n if case["rows_form"] else n * d
        return {"bytes": 2.0 * passes * n * d * es, "flops": passes * (n * d + mask * drawn)}
    k = case["rows"]
    tokens = n * (4 if case["index"] == "i32" else 8)
    if case["op"] == "lookup":
        return {"bytes": float(tokens + min(n, k) * d * es + n * d * es),
                "flops": n * d * (1.0 + mask)}
    if case["op"] == "gradient":
        return {"bytes": float(tokens + n * d * es + k * d * es), "flops": n * d * (1.0 + mask)}
    return {"bytes": float(tokens + n * d * es + 24 * k * d),
            "flops": n * d * (1.0 + mask) + 14.0 * k * d}


# ---------------------------------------------------------------------------
# The definition in 64 bits.

def _exact_words(count, seed, offset):
    """The generator's words of the first `count` elements, from products in
    16-bit halves."""

    def product(x, m):
        low, high = x & 0xFFFF, x >> 16
        ml, mh = m & 0xFFFF, m >> 16
        ll, lh, hl = low * ml, low * mh, high * ml
        middle = (ll >> 16) + (lh & 0xFFFF) + (hl & 0xFFFF)
        return (high * mh + (lh >> 16) + (hl >> 16) + (middle >> 16),
                ((middle & 0xFFFF) << 16) | (ll & 0xFFFF))

    blocks = torch.arange(-(-count // 4), dtype=torch.int64, device="cuda")
    x = [blocks % 2 ** 32, blocks // 2 ** 32, torch.full_like(blocks, offset % 2 ** 32),
         torch.full_like(blocks, offset // 2 ** 32)]
    key = [seed % 2 ** 32, seed // 2 ** 32]
    for _ in range(10):
        high0, low0 = product(x[0], 0xD2511F53)
        high1, low1 = product(x[2], 0xCD9E8D57)
        x = [high1 ^ x[1] ^ key[0], low1, high0 ^ x[3] ^ key[1], low0]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    out = torch.empty(4 * len(blocks), dtype=torch.int64, device="cuda")
    for j in range(4):
        out[j::4] = x[j]
    return out[:count]


def exact(case, seed):
    s = _inputs(case, seed)
    n, d, p = case["tokens"], case["width"], case["p"]
    if p > 0:
        by_row = case["op"] == "dropout" and case["rows_form"]
        words = _exact_words(n if by_row else n * d, s["seed"], s["offset"])
        weight = (words >= math.floor(p * 2 ** 32)).double() / (1.0 - p)
        weight = weight.view(n, 1) if by_row else weight.view(n, d)
    else:
        weight = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    if case["op"] == "dropout":
        y = s["x"].double() * weight
        return {"y": y, "dx": s["grad"].double() * weight} if case["backward"] else y
    weight = weight * case["scale"]
    index = s["index"].long()
    named = (index >= 0).nonzero().view(-1)
    if case["op"] == "lookup":
        y = torch.zeros(n, d, dtype=torch.float64, device="cuda")
        y[named] = s["table"].double().index_select(0, index[named])
        return y * weight
    terms = (s["grad"].double() * weight)[named]
    total = torch.zeros(case["rows"], d, dtype=torch.float64, device="cuda")
    total.index_put_((index[named],), terms, accumulate=True)
    if case["op"] == "gradient":
        return total
    first = 0.9 * s["first"].double() + 0.1 * total
    second = 0.999 * s["second"].double() + 0.001 * total ** 2
    table = s["table"].double() - RATE / BIAS1 * first / (torch.sqrt(second) / BIAS2_SQRT + EPS)
    return {"table": table, "first": first, "second": second}
