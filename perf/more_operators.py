"""Cases for the operators around a paged cache that several sequences share: rotary positions, the cache written and read back, attention over a prefix
that many sequences have in common.

The model behind the sizes is the 27B hybrid of the library's headers: 24 query heads over 4 kv heads of 256, the first 64 dims rotated, K/V cache in Q8_0,
pages of 64 positions.

  rope    queries and keys turned by their positions: halves or neighbours paired, part of the head, frequencies scaled for long contexts
  write   norms and rotation of queries and keys, the keys and the values quantised into the cache
  read    rows of the cache back as floats
  shared  attention of the new tokens of groups of sequences, each group over pages that it has in common and over each sequence's own

A case's lists are texts, numbers separated by commas.  `own` chooses between the library's entry points and plain torch operations.
"""
import math
import os
import sys

import torch

own = False

N_HEAD, N_HEAD_KV, HEAD_DIM, N_ROT, THETA, TRAINED = 24, 4, 256, 64, 1e7, 262144
GROUP = N_HEAD // N_HEAD_KV
PAGE, BLOCK, BLOCKS = 64, 34, HEAD_DIM // 32       # positions of a page; bytes of a Q8_0 block (fp16 scale, 32 codes), blocks of a row
EPS = 1e-6
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _bb():
    path = os.path.join(os.getcwd(), "p40-kernel_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import bonsai_b200
    return bonsai_b200


def listed():
    return [
        # one decoded token: a latency
        {"name": "rope 1 token", "op": "rope", "n_tok": 1, "heads": N_HEAD, "heads_kv": N_HEAD_KV, "dim": HEAD_DIM, "n_rot": N_ROT, "next": 0, "factor": 1},
        # a chunk of a prompt of a model with neighbouring pairs and whole heads turned, four times beyond what it was trained for
        {"name": "rope 2999 tokens, neighbours, scaled", "op": "rope", "n_tok": 2999, "heads": 32, "heads_kv": 8, "dim": 128, "n_rot": 128, "next": 1, "factor": 4},
        # one decoded token of each of 16 chats of different age
        {"name": "write 16 sequences, 1 token each", "op": "write", "norm": 1, "next": 0, "factor": 1,
         "cached": "40,1800,1000,63,64,700,500,1047,129,330,1500,0,900,601,250,311", "new": ",".join(["1"] * 16)},
        # a chunk of a prompt
        {"name": "write 2000 tokens", "op": "write", "norm": 1, "next": 0, "factor": 4, "cached": "1000", "new": "2000"},
        # what is left of a context whose oldest part is dropped, to be turned back and written again
        {"name": "read 700 rows, fp32", "op": "read", "first": "1301", "rows": "700", "type": "fp32"},
        # two contexts kept in another form
        {"name": "read 30000 and 5003 rows, bf16", "op": "read", "first": "0,100", "rows": "30000,5003", "type": "bf16"},
        # 16 answers to one long prompt, all young
        {"name": "shared 16 answers over 8192", "op": "shared", "groups": "16", "shared": "128",
         "cached": "0,5,17,30,64,100,128,150,200,220,255,256,300,320,350,400", "new": ",".join(["1"] * 16)},
        # chats of different age behind one instruction
        {"name": "shared 64 chats behind 2048", "op": "shared", "groups": "64", "shared": "32",
         "cached": ",".join(str(37 * i * i % 1500) for i in range(64)), "new": ",".join(["1"] * 64)},
        # four answers with five drafted tokens each to verify, late in a long context
        {"name": "shared 4 x 5 drafted tokens at 32000", "op": "shared", "groups": "4", "shared": "500", "cached": "10,70,0,133", "new": "5,5,5,5"},
        # many samples of one prompt
        {"name": "shared 200 answers over 16000", "op": "shared", "groups": "200", "shared": "250",
         "cached": ",".join(str(i % 61) for i in range(200)), "new": ",".join(["1"] * 200)},
        # questions of one document
        {"name": "shared 12 questions behind 6016", "op": "shared", "groups": "12", "shared": "94", "cached": ",".join(["0"] * 12),
         "new": "20,35,150,64,7,91,48,33,120,15,77,40"},
        # a serving step: two documents with chats, prompts and one that pauses, and two that share nothing
        {"name": "shared ragged batch", "op": "shared", "groups": "5,3,1,1", "shared": "47,16,0,0",
         "cached": "0,100,700,31,64,0,2000,10,1500,0", "new": "1,30,1,0,5,200,1,1,1,300"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def draw(rng):
    op = rng.choice(["rope", "write", "read", "shared", "shared", "shared", "shared"])
    if op == "rope":
        dim = rng.choice([64, 80, 128, 256])
        heads_kv = rng.choice([1, 2, 4, 8])
        return {"op": op, "n_tok": _log_int(rng, 1, 2900), "heads": heads_kv * rng.choice([1, 2, 4]), "heads_kv": heads_kv, "dim": dim,
                "n_rot": rng.choice([dim, dim // 2, dim // 4]), "next": rng.choice([0, 1]), "factor": rng.choice([1, 2, 4, 8])}
    if op == "write":
        n_seq = _log_int(rng, 1, 16)
        return {"op": op, "norm": rng.choice([0, 1]), "next": rng.choice([0, 1]), "factor": rng.choice([1, 4]),
                "cached": _text([rng.choice([0, _log_int(rng, 1, 2000)]) for _ in range(n_seq)]), "new": _text([_log_int(rng, 1, 1900 // n_seq) for _ in range(n_seq)])}
    if op == "read":
        n_seq, kind = _log_int(rng, 1, 6), rng.choice(["fp32", "fp16", "bf16"])
        most = (20000 if kind == "fp32" else 34000) // n_seq
        return {"op": op, "first": _text([rng.choice([0, _log_int(rng, 1, 3000)]) for _ in range(n_seq)]),
                "rows": _text([_log_int(rng, 1, most) for _ in range(n_seq)]), "type": kind}
    left, rows, groups, shared, cached, new = 4_000_000, 50_000, [], [], [], []      # pairs of a token and a position; positions
    for _ in range(_log_int(rng, 1, 4)):
        n_seq = _log_int(rng, 1, 64)
        pages = _log_int(rng, 1, 300)
        kind, fit = rng.random(), 0
        for _ in range(n_seq):
            c = rng.choice([0, _log_int(rng, 1, 1500)])
            n = 1 if kind < 0.5 else _log_int(rng, 1, 8) if kind < 0.8 else _log_int(rng, 1, 150)
            if fit and (n * (PAGE * pages + c + n) > left or c + n > rows):
                break
            left -= n * (PAGE * pages + c + n)
            rows -= c + n
            fit += 1
            cached.append(c)
            new.append(n)
        groups.append(fit)
        shared.append(pages)
    return {"op": op, "groups": _text(groups), "shared": _text(shared), "cached": _text(cached), "new": _text(new)}


# ---- inputs ------------------------------------------------------------------------------------------
def _starts(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return at


def _i32(numbers):
    return torch.tensor(numbers, dtype=torch.int32, device="cuda")


def _rounded_away(x):
    """To the nearest whole number, halves away from zero (|x| < 2^23, fp32)."""
    return torch.trunc(x + torch.copysign(torch.full_like(x, 0.49999997), x))


def _half_away(x):
    """Values >= 0 to fp16, halves away from zero, as fp32."""
    x = x.double()
    e = torch.clamp(torch.frexp(x)[1] - 1, min=-14)
    step = torch.ldexp(torch.ones_like(x), e - 10)
    return (torch.floor(x / step + 0.5) * step).float()


def _q8_0(x):
    """Rows of blocks of 32 -> codes (whole numbers, fp32) and scales (fp16 values, fp32): [..., blocks, 32], [..., blocks].  The scale is the largest
    magnitude times 1 / 127, rounded once, in fp32."""
    x = x.reshape(*x.shape[:-1], -1, 32)
    d = x.abs().amax(-1) * torch.full((), 1 / 127, dtype=torch.float32, device=x.device)
    inv = torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
    return _rounded_away(x * inv[..., None]).clamp(-127, 127), _half_away(d)


def _blocks(x):
    """Q8_0 blocks of the rows x, as bytes [..., blocks, 34]."""
    codes, scale = _q8_0(x)
    return torch.cat([scale.half()[..., None].contiguous().view(torch.uint8), codes.to(torch.int8).view(torch.uint8)], -1)


def _scaled(n_rot, theta, factor):
    """Radians per position of the pairs, and what turned values are multiplied by.  Beyond factor 1, as a model that was trained for TRAINED positions is
    taken to factor times as many: pairs that turn more than 32 times in TRAINED keep their frequency, those that turn less than once are slowed by the
    factor, the ones between by a part of it that grows with their number."""
    pairs = n_rot // 2
    freq = [theta ** (-i / pairs) for i in range(pairs)]
    if factor == 1:
        return freq, 1.0
    at = lambda turns: n_rot * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    low, high = max(0, math.floor(at(32))), min(n_rot - 1, math.ceil(at(1)))
    slowed = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(pairs)]
    return [f * (1 - s) + f / factor * s for f, s in zip(freq, slowed)], 0.1 * math.log(factor) + 1


def _rotation(s, g, n_rot, n_tok, factor):
    freq, amplitude = _scaled(n_rot, THETA, factor)
    s.update(freq=torch.tensor(freq, dtype=torch.float64, device="cuda"), amplitude=float(torch.tensor(amplitude, dtype=torch.float32)))


def _filled(pages, g):
    """One layer's pages with rows of a normal distribution, some heads and some positions larger than others."""
    pool = torch.empty(pages, 1, 2, N_HEAD_KV, PAGE, BLOCKS, BLOCK, dtype=torch.uint8, device="cuda")
    for p in range(0, pages, 64):
        rows = torch.randn(*pool[p:p + 64].shape[:5], HEAD_DIM, generator=g, device="cuda")
        pool[p:p + 64] = _blocks(rows * torch.exp(0.3 * torch.randn(*rows.shape[:5], 1, generator=g, device="cuda")))
    return pool


def _tables(used, g):
    """Pages of sequences that share none, in any order: [sequences][most pages], and how many there are."""
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device="cuda")
    table, at = torch.zeros(len(used), max(max(used), 1), dtype=torch.int32, device="cuda"), 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    return table, pages


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s, op = dict(case), case["op"]
    if op == "rope":
        n, dim = case["n_tok"], case["dim"]
        s.update(q=normal(n, case["heads"], dim) * 2, k=normal(n, case["heads_kv"], dim) * 2, pos=torch.arange(n, dtype=torch.int32, device="cuda") + 1000 * (1 + seed % 200),
                 q_out=torch.empty(n, case["heads"], dim, device="cuda"), k_out=torch.empty(n, case["heads_kv"], dim, device="cuda"))
        _rotation(s, g, case["n_rot"], n, case["factor"])
        return s
    if op == "read":
        first, rows = _ints(case["first"]), _ints(case["rows"])
        length = [f + n for f, n in zip(first, rows)]
        table, pages = _tables([-(-c // PAGE) for c in length], g)
        n = sum(rows)
        out = lambda: torch.empty(n, N_HEAD_KV, HEAD_DIM, dtype=TYPES[case["type"]], device="cuda")  # noqa: E731
        s.update(pool=_filled(pages, g), table=table, k_out=out(), v_out=out(), first_dev=_i32(first))
        seq = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), torch.tensor(rows, device="cuda"))
        s["seq"], s["pos"] = seq, torch.arange(n, device="cuda") + (s["first_dev"] - _i32(_starts(rows))[:-1])[seq]
        if own:
            s["cache"] = _bb().Pages(s["pool"], table, _i32(length), _i32(_starts(rows)), 1, N_HEAD_KV, n)
        return s
    cached, new = _ints(case["cached"]), _ints(case["new"])
    n = sum(new)
    if op == "write":
        length = [c + m for c, m in zip(cached, new)]
        table, pages = _tables([-(-c // PAGE) for c in length], g)
        # q is half of its projection's rows, the other half gates the output
        s.update(pool=_filled(pages, g), table=table, proj=normal(n, N_HEAD, 2 * HEAD_DIM) * 2, k=normal(n, N_HEAD_KV, HEAD_DIM) * 2, v=normal(n, N_HEAD_KV, HEAD_DIM),
                 q_weight=1 + 0.1 * normal(HEAD_DIM), k_weight=1 + 0.1 * normal(HEAD_DIM), q_out=torch.empty(n, N_HEAD, HEAD_DIM, device="cuda"))
        _rotation(s, g, N_ROT, n, case["factor"])
        seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
        s["seq"], s["pos"] = seq, torch.arange(n, device="cuda") + (_i32(length) - _i32(_starts(new))[1:])[seq]
        if own:
            s["cache"] = _bb().Pages(s["pool"], table, _i32(length), _i32(_starts(new)), 1, N_HEAD_KV, n)
        return s
    groups, shared = _ints(case["groups"]), _ints(case["shared"])
    of = [i for i, m in enumerate(groups) for _ in range(m)]
    length = [PAGE * shared[of[i]] + c + m for i, (c, m) in enumerate(zip(cached, new))]
    used = [-(-c // PAGE) for c in length]
    pages = sum(shared) + sum(u - shared[of[i]] for i, u in enumerate(used)) + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table, at, common = torch.zeros(len(new), max(max(used), 1), dtype=torch.int32, device="cuda"), 0, []
    for m in shared:
        common.append(order[at:at + m])
        at += m
    for i, u in enumerate(used):
        m = shared[of[i]]
        table[i, :m] = common[of[i]]
        table[i, m:u] = order[at:at + u - m]
        at += u - m
    s.update(pool=_filled(pages, g), table=table, lengths=length, starts=_starts(new), firsts=_starts(groups), pages=shared, q=normal(n, N_HEAD, HEAD_DIM),
             out=torch.empty(n, N_HEAD, HEAD_DIM, device="cuda"))
    if own:
        bb = _bb()
        s["cache"] = bb.Pages(s["pool"], table, _i32(length), _i32(_starts(new)), 1, N_HEAD_KV, n)
        s["group"], s["shared_dev"] = _i32(_starts(groups)), _i32(shared)
        s["workspace"] = torch.empty(max(1, s["cache"].attn_shared_workspace(len(groups), N_HEAD)), dtype=torch.uint8, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------------------
def _ok(rc):
    if rc != 0:
        raise RuntimeError("the library returned %d" % rc)


def run(s):
    return {"rope": _run_rope, "write": _run_write, "read": _run_read, "shared": _run_shared}[s["op"]](s)


def _turned(x, s, n_rot):
    """Rows [tokens, heads, dim] by the tokens' positions."""
    angle = s["pos"].double()[:, None] * s["freq"]
    c, d = ((f(angle) * s["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    if s["next"]:
        a, b = x[..., 0:n_rot:2], x[..., 1:n_rot:2]
        return torch.cat([torch.stack([a * c - b * d, b * c + a * d], -1).flatten(-2), x[..., n_rot:]], -1)
    a, b = x[..., :n_rot // 2], x[..., n_rot // 2:n_rot]
    return torch.cat([a * c - b * d, b * c + a * d, x[..., n_rot:]], -1)


def _run_rope(s):
    if own:
        h, hk, dim = s["heads"], s["heads_kv"], s["dim"]
        _ok(_bb().rope(s["q"], s["k"], s["pos"], s["freq"], s["q_out"], s["k_out"], s["n_tok"], h, hk, dim, s["n_rot"], s["next"], s["amplitude"],
                       h * dim, dim, hk * dim, dim))
        return [s["q_out"], s["k_out"]]
    return [_turned(s["q"], s, s["n_rot"]), _turned(s["k"], s, s["n_rot"])]


def _parts(pool):
    """What the cache's bytes stand for: codes and scales."""
    return [pool[..., 2:].view(torch.int8), pool[..., :2].view(torch.float16)]


def _run_write(s):
    if own:
        w = (s["q_weight"], s["k_weight"]) if s["norm"] else (None, None)
        d = HEAD_DIM
        _ok(s["cache"].write(0, s["proj"], s["k"], s["v"], *w, None, s["freq"], s["q_out"], N_HEAD, N_ROT, s["next"], s["amplitude"],
                             N_HEAD * 2 * d, 2 * d, N_HEAD_KV * d, d, N_HEAD_KV * d, d, EPS))
        return [s["q_out"], *_parts(s["pool"])]

    def rows(x, w):
        if s["norm"]:       # the mean and its root in 64 bits: codes lie next to borders
            x = x * (1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + EPS)).float() * w
        return _turned(x, s, N_ROT)
    q = rows(s["proj"][..., :HEAD_DIM], s["q_weight"])
    page, at = s["table"][s["seq"], s["pos"] // PAGE].long(), s["pos"] % PAGE
    for i, x in enumerate((rows(s["k"], s["k_weight"]), s["v"])):
        s["pool"][page, 0, i, :, at] = _blocks(x)
    return [q, *_parts(s["pool"])]


def _run_read(s):
    if own:
        _ok(s["cache"].read(0, s["first_dev"], s["k_out"], s["v_out"]))
        return [s["k_out"], s["v_out"]]
    page, at = s["table"][s["seq"], s["pos"] // PAGE].long(), s["pos"] % PAGE
    rows = [s["pool"][page, 0, i, :, at] for i in range(2)]
    return [(x[..., 2:].view(torch.int8).float() * x[..., :2].view(torch.float16).float()).flatten(-2).to(TYPES[s["type"]]) for x in rows]


def _floats(s, pages):
    """K and V of these pages, [kv heads, positions, dims] each."""
    held = s["pool"][pages.long(), 0]                                                     # pages, K | V, kv heads, positions, blocks, bytes
    held = held[..., 2:].view(torch.int8).float() * held[..., :2].view(torch.float16).float()
    return held.permute(1, 2, 0, 3, 4, 5).reshape(2, N_HEAD_KV, -1, HEAD_DIM)


def _part(q, k, v, seen=None):
    """Largest score, sum of weights and sum of weighted values of the rows q [tokens, kv heads, group, dims]."""
    score = torch.einsum("thgd,hpd->htgp", q, k) * HEAD_DIM ** -0.5
    if seen is not None:
        score = torch.where(seen[:, None], score, -math.inf)
    m = score.amax(-1, keepdim=True)
    p = torch.exp(score - m)
    return m, p.sum(-1, keepdim=True), torch.einsum("htgp,hpd->htgd", p, v)


def _run_shared(s):
    if own:
        _ok(s["cache"].attn_shared(0, s["group"], s["shared_dev"], s["q"], s["out"], N_HEAD, s["workspace"], HEAD_DIM ** -0.5))
        return s["out"]
    codes, d = _q8_0(s["q"])
    q = (codes * d[..., None]).reshape(-1, N_HEAD_KV, GROUP, HEAD_DIM)
    for g, m in enumerate(s["pages"]):
        first, last = s["firsts"][g:g + 2]
        a, b = s["starts"][first], s["starts"][last]
        if a == b:
            continue
        if m:
            shared = _part(q[a:b], *_floats(s, s["table"][first, :m]))
        for i in range(first, last):
            lo, hi = s["starts"][i:i + 2]
            if lo == hi:
                continue
            n = s["lengths"][i] - PAGE * m
            k, v = _floats(s, s["table"][i, m:m - (-n // PAGE)])
            seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - (hi - lo), n, device="cuda")[:, None]
            top, total, o = _part(q[lo:hi], k[:, :n], v[:, :n], seen)
            if m:
                top2, total2, o2 = (x[:, lo - a:hi - a] for x in shared)
                most = torch.maximum(top, top2)
                f, f2 = torch.exp(top - most), torch.exp(top2 - most)
                total, o = total * f + total2 * f2, o * f + o2 * f2
            s["out"][lo:hi] = (o / total).transpose(0, 1).reshape(hi - lo, N_HEAD, HEAD_DIM)
    return s["out"]


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    """Every input read once, every output written once; two operations per product.  A cache's pages are read where a new token sees them, shared ones once."""
    op, row = case["op"], BLOCKS * BLOCK
    if op == "rope":
        n, heads = case["n_tok"], case["heads"] + case["heads_kv"]
        return {"bytes": n * heads * case["dim"] * 8 + 4 * n + 4 * case["n_rot"], "flops": n * heads * case["n_rot"] * 3}
    if op == "read":
        return {"bytes": sum(_ints(case["rows"])) * N_HEAD_KV * 2 * (row + HEAD_DIM * (4 if case["type"] == "fp32" else 2)), "flops": sum(_ints(case["rows"])) * N_HEAD_KV * 2 * HEAD_DIM}
    cached, new = _ints(case["cached"]), _ints(case["new"])
    n = sum(new)
    if op == "write":
        return {"bytes": n * (N_HEAD * HEAD_DIM * 8 + N_HEAD_KV * (HEAD_DIM * 8 + 2 * row)), "flops": n * ((N_HEAD + N_HEAD_KV) * (4 * HEAD_DIM + 3 * N_ROT) + N_HEAD_KV * 6 * HEAD_DIM)}
    of = [i for i, m in enumerate(_ints(case["groups"])) for _ in range(m)]
    before = [PAGE * _ints(case["shared"])[g] for g in of]
    rows = sum(PAGE * m for g, m in enumerate(_ints(case["shared"])) if any(new[i] for i in range(len(new)) if of[i] == g)) + sum(c + m for c, m in zip(cached, new) if m)
    pairs = sum(m * (p + c) + m * (m + 1) // 2 for p, c, m in zip(before, cached, new))
    return {"bytes": 2 * N_HEAD_KV * row * rows + n * N_HEAD * HEAD_DIM * 8, "flops": 4 * HEAD_DIM * N_HEAD * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]

    def turned(x, n_rot):
        x = x.double()
        spin = torch.polar(torch.full_like(s["freq"], s["amplitude"]), s["pos"].double()[:, None] * s["freq"])[:, None]
        if s["next"]:
            z = torch.view_as_complex(x[..., :n_rot].reshape(*x.shape[:-1], -1, 2).contiguous()) * spin
            return torch.cat([torch.view_as_real(z).flatten(-2), x[..., n_rot:]], -1)
        z = torch.complex(x[..., :n_rot // 2], x[..., n_rot // 2:n_rot]) * spin
        return torch.cat([z.real, z.imag, x[..., n_rot:]], -1)

    if op == "rope":
        return [turned(s["q"], case["n_rot"]), turned(s["k"], case["n_rot"])]
    if op == "write":
        x = s["proj"][..., :HEAD_DIM].double()
        if case["norm"]:
            x = s["q_weight"].double() * x * ((x ** 2).sum(-1, keepdim=True) / HEAD_DIM + EPS) ** -0.5
        return [turned(x, N_ROT), None, None]
    number = lambda rows: (rows[..., 2:].view(torch.int8).double() * rows[..., :2].view(torch.float16).double()).flatten(-2)  # noqa: E731
    if op == "read":
        # token by token of a sequence, through its table
        out = [torch.empty(s["k_out"].shape, dtype=torch.float64, device="cuda") for _ in range(2)]
        at = 0
        for i, (f, n) in enumerate(zip(_ints(case["first"]), _ints(case["rows"]))):
            for j in range(2):
                whole = number(s["pool"][s["table"][i].long(), 0, j]).transpose(1, 2).flatten(0, 1)      # positions, kv heads, dims
                out[j][at:at + n] = whole[f:f + n]
            at += n
        return out
    out = torch.zeros_like(s["out"], dtype=torch.float64)
    q = number(_blocks(s["q"]))
    for i, (lo, hi) in enumerate(zip(s["starts"], s["starts"][1:])):
        c = s["lengths"][i]
        for h in range(N_HEAD_KV if hi > lo else 0):
            k, v = (number(s["pool"][s["table"][i].long(), 0, j, h]).flatten(0, 1)[:c] for j in range(2))
            score = q[lo:hi, h * GROUP:(h + 1) * GROUP] @ k.T / math.sqrt(HEAD_DIM)
            hidden = torch.ones(hi - lo, c, dtype=torch.bool, device="cuda").triu(c - (hi - lo) + 1)
            out[lo:hi, h * GROUP:(h + 1) * GROUP] = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), -1) @ v
    return out
