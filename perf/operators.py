"""Cases for the operators that a layer needs between its projections when a program serves prompts and several sequences.

The model behind the sizes is the 27B hybrid of the library's headers: 16 attention layers (24 query heads over 4 kv heads of
256, the first 64 dims rotated, K/V cache in Q8_0), 48 delta-net layers (16 key heads, 48 value heads, [128][128] state each).

  qk      norms of queries and keys for each head, with the position rotation
  attend  the K and V rows of new tokens into a paged cache, and their attention over it, for several sequences
  copy    pages copied inside a cache: a fork's last page, a compaction
  delta   the gated delta rule over the tokens of several sequences

A case's lists (new tokens, cached positions of each sequence) are texts, numbers separated by commas.  `own` chooses
between the library's entry points and plain torch operations.
"""
import math
import os
import sys

import torch

own = False

N_HEAD, N_HEAD_KV, HEAD_DIM, N_ROT, THETA = 24, 4, 256, 64, 1e7
GROUP = N_HEAD // N_HEAD_KV
KV_LAYERS = 16
PAGE, BLOCK, BLOCKS = 64, 34, HEAD_DIM // 32       # positions of a page; bytes of a Q8_0 block (fp16 scale, 32 codes), blocks of a row
GDN_K_HEADS, GDN_V_HEADS, GDN_DIM = 16, 48, 128
EPS = 1e-6


def _bb():
    path = os.path.join(os.getcwd(), "p40-kernel_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import bonsai_b200
    return bonsai_b200


def listed():
    return [
        # one decoded token of one sequence: a latency
        {"name": "qk 1 token", "op": "qk", "n_tok": 1},
        # a chunk of a prompt far into a long context; q is half of the projection's rows, the other half gates the output
        {"name": "qk 2000 tokens", "op": "qk", "n_tok": 2000},
        # one decoded token of each of 16 chats of different age
        {"name": "attend 16 sequences, 1 token each", "op": "attend", "layers": 1,
         "cached": "40,8000,1000,63,64,700,5000,2047,129,3300,1500,0,900,6001,2500,311", "new": ",".join(["1"] * 16)},
        # five drafted tokens to verify late in a long context
        {"name": "attend 5 drafted tokens at 32700", "op": "attend", "layers": 1, "cached": "32700", "new": "5"},
        # a chunk of a prompt behind what earlier chunks left
        {"name": "attend 512 tokens after 4000", "op": "attend", "layers": 1, "cached": "4000", "new": "512"},
        # a serving step: a fresh prompt, the ends of two others, two decoding sequences and one that pauses
        {"name": "attend ragged batch", "op": "attend", "layers": 2, "cached": "0,1000,63,64,2500,900", "new": "700,1,65,1,200,0"},
        # copy on write: the last page of a chat that four answers continue
        {"name": "copy fork of 4 pages", "op": "copy", "pages": 64, "moved": 4},
        # the pages in use moved to the front of the pool
        {"name": "copy compaction of 300 pages", "op": "copy", "pages": 700, "moved": 300},
        # one decoded token of each of 16 chats
        {"name": "delta 16 sequences, 1 token each", "op": "delta", "new": ",".join(["1"] * 16)},
        # four drafted tokens of three chats
        {"name": "delta 3 sequences, 4 drafted tokens", "op": "delta", "new": "4,4,4"},
        # a prompt
        {"name": "delta 2048 tokens", "op": "delta", "new": "2048"},
        # a serving step
        {"name": "delta ragged batch", "op": "delta", "new": "700,1,65,1,200,0"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def draw(rng):
    op = rng.choice(["qk", "attend", "attend", "attend", "copy", "delta", "delta"])
    if op == "qk":
        return {"op": op, "n_tok": _log_int(rng, 1, 1999)}
    if op == "copy":
        moved = _log_int(rng, 1, 299)
        return {"op": op, "pages": moved + _log_int(rng, moved, 400), "moved": moved}
    n_seq = _log_int(rng, 1, 16)
    if op == "delta":
        if rng.random() < 0.4:      # a decoding step
            return {"op": op, "new": _text([_log_int(rng, 1, 16) for _ in range(n_seq)])}
        left, new = _log_int(rng, 17, 2047), []
        for _ in range(n_seq):
            new.append(min(left, _log_int(rng, 1, 1500)))
            left -= new[-1]
        return {"op": op, "new": _text(new)}
    if rng.random() < 0.5:          # a decoding step, drafted tokens or not
        cached = [_log_int(rng, 1, 40000 // n_seq) for _ in range(n_seq)]
        new = [_log_int(rng, 1, 8) if rng.random() < 0.5 else 1 for _ in range(n_seq)]
        return {"op": op, "layers": 1, "cached": _text(cached), "new": _text(new)}
    pairs, cached, new = 2_200_000, [], []      # prompts
    for _ in range(min(n_seq, 6)):
        c, n = rng.choice([0, _log_int(rng, 1, 6000)]), _log_int(rng, 2, 600)
        n = max(0, min(n, pairs // (c + n)))
        pairs -= n * (c + n)
        cached.append(c)
        new.append(n)
    return {"op": op, "layers": 1, "cached": _text(cached), "new": _text(new)}


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
    """Rows of blocks of 32 -> codes (whole numbers, fp32) and scales (fp16 values, fp32): [..., blocks, 32], [..., blocks]."""
    x = x.reshape(*x.shape[:-1], -1, 32)
    d = x.abs().amax(-1) / 127.0
    inv = torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
    return _rounded_away(x * inv[..., None]).clamp(-127, 127), _half_away(d)


def _blocks(x):
    """Q8_0 blocks of the rows x, as bytes [..., blocks, 34]."""
    codes, scale = _q8_0(x)
    return torch.cat([scale.half()[..., None].contiguous().view(torch.uint8), codes.to(torch.int8).view(torch.uint8)], -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s, op = dict(case), case["op"]
    if op == "qk":
        n = case["n_tok"]
        s.update(proj=normal(n, N_HEAD, 2 * HEAD_DIM) * 2, k=normal(n, N_HEAD_KV, HEAD_DIM) * 2,
                 q_weight=1 + 0.1 * normal(HEAD_DIM), k_weight=1 + 0.1 * normal(HEAD_DIM),
                 pos=torch.arange(n, dtype=torch.int32, device="cuda") + 1000 * (1 + seed % 200),
                 freq=THETA ** (-torch.arange(N_ROT // 2, dtype=torch.float64, device="cuda") / (N_ROT // 2)),
                 q_out=torch.empty(n, N_HEAD, HEAD_DIM, device="cuda"), k_out=torch.empty(n, N_HEAD_KV, HEAD_DIM, device="cuda"))
    elif op == "copy":
        n, m = case["pages"], case["moved"]
        rows = torch.randint(0, 256, (n, KV_LAYERS, 2, N_HEAD_KV, PAGE, BLOCKS * BLOCK), generator=g, device="cuda", dtype=torch.uint8)
        order = torch.randperm(n, generator=g, device="cuda")
        src, dst = order[:m].sort().values, order[m:2 * m].sort().values
        s.update(pool=rows, src=src, dst=dst, src_host=src.int().cpu(), dst_host=dst.int().cpu())
    elif op == "attend":
        cached, new, layers = _ints(case["cached"]), _ints(case["new"]), case["layers"]
        length = [c + n for c, n in zip(cached, new)]
        used = [-(-c // PAGE) for c in length]
        wide = max(max(used), 1)
        pages = sum(used) + 3
        order = torch.randperm(pages, generator=g, device="cuda")
        table, at = torch.zeros(len(new), wide, dtype=torch.int32, device="cuda"), 0
        for i, u in enumerate(used):
            table[i, :u] = order[at:at + u]
            at += u
        pool = torch.empty(pages, layers, 2, N_HEAD_KV, PAGE, BLOCKS, BLOCK, dtype=torch.uint8, device="cuda")
        for p in range(0, pages, 64):
            pool[p:p + 64] = _blocks(normal(*pool[p:p + 64].shape[:5], HEAD_DIM))
        n = sum(new)
        s.update(pool=pool, table=table, length=_i32(length), start=_i32(_starts(new)), lengths=length, starts=_starts(new), max_len=max(length),
                 q=normal(layers, n, N_HEAD, HEAD_DIM), k=normal(layers, n, N_HEAD_KV, HEAD_DIM), v=normal(layers, n, N_HEAD_KV, HEAD_DIM),
                 out=torch.empty(layers, n, N_HEAD, HEAD_DIM, device="cuda"))
        # where each new row goes
        seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
        s["seq"], s["pos"] = seq, torch.arange(n, device="cuda") + (s["length"] - s["start"][1:])[seq]
        if own:
            bb = _bb()
            s["cache"] = bb.Pages(pool, table, s["length"], s["start"], layers, N_HEAD_KV, n)
            s["workspace"] = torch.empty(max(1, bb.pages_attn_workspace(n, max(length), len(new), N_HEAD, N_HEAD_KV)), dtype=torch.uint8, device="cuda")
    else:
        new = _ints(case["new"])
        n, unit = sum(new), lambda x: x / x.norm(dim=-1, keepdim=True)
        # the decays of a trained model lie between some that forget at once and some that hardly forget
        speed = torch.exp(normal(GDN_V_HEADS) * 1.5 - 2)
        s.update(state=normal(len(new), GDN_V_HEADS, GDN_DIM, GDN_DIM) * 0.1, q=unit(normal(n, GDN_K_HEADS, GDN_DIM)) * GDN_DIM ** -0.5,
                 k=unit(normal(n, GDN_K_HEADS, GDN_DIM)), v=normal(n, GDN_V_HEADS, GDN_DIM),
                 g=-speed * torch.nn.functional.softplus(normal(n, GDN_V_HEADS)), beta=torch.sigmoid(normal(n, GDN_V_HEADS)),
                 out=torch.empty(n, GDN_V_HEADS, GDN_DIM, device="cuda"), start=_i32(_starts(new)), starts=_starts(new))
        if own:
            size = _bb().gdn_seqs_workspace(n, len(new), GDN_K_HEADS, GDN_V_HEADS, GDN_DIM, GDN_DIM)
            s["workspace"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------------------
def _ok(rc):
    if rc != 0:
        raise RuntimeError("the library returned %d" % rc)


def run(s):
    return {"qk": _run_qk, "attend": _run_attend, "copy": _run_copy, "delta": _run_delta}[s["op"]](s)


def _run_qk(s):
    n = s["n_tok"]
    if own:
        _ok(_bb().qk_norm_rope(s["proj"], s["k"], s["q_weight"], s["k_weight"], s["pos"], s["freq"], s["q_out"], s["k_out"], n, N_HEAD, N_HEAD_KV,
                               HEAD_DIM, N_ROT, N_HEAD * 2 * HEAD_DIM, 2 * HEAD_DIM, N_HEAD_KV * HEAD_DIM, HEAD_DIM, EPS))
        return [s["q_out"], s["k_out"]]
    angle = s["pos"].double()[:, None] * s["freq"]
    c, d = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., :N_ROT // 2], x[..., N_ROT // 2:N_ROT]
        return torch.cat([a * c - b * d, b * c + a * d, x[..., N_ROT:]], -1)
    return [turned(s["proj"][..., :HEAD_DIM], s["q_weight"]), turned(s["k"], s["k_weight"])]


def _parts(pool):
    """What the cache's bytes stand for: codes and scales."""
    return [pool[..., 2:].view(torch.int8), pool[..., :2].view(torch.float16)]


def _run_attend(s):
    scale = HEAD_DIM ** -0.5
    if own:
        for layer in range(s["layers"]):
            _ok(s["cache"].append(layer, s["k"][layer], s["v"][layer]))
            _ok(s["cache"].attn(layer, s["q"][layer], s["out"][layer], N_HEAD, s["max_len"], s["workspace"], scale))
        return [s["out"], *_parts(s["pool"])]
    page, at = s["table"][s["seq"], s["pos"] // PAGE].long(), s["pos"] % PAGE
    for layer in range(s["layers"]):
        for i, rows in enumerate((s["k"][layer], s["v"][layer])):
            s["pool"][page, layer, i, :, at] = _blocks(rows)
        codes, d = _q8_0(s["q"][layer])
        q = (codes * d[..., None]).reshape(-1, N_HEAD_KV, GROUP, HEAD_DIM)
        for i, n in enumerate(s["lengths"]):
            lo, hi = s["starts"][i:i + 2]
            if hi == lo:
                continue
            held = s["pool"][s["table"][i, :-(-n // PAGE)].long(), layer]                   # pages, K | V, kv heads, positions, blocks, bytes
            held = held[..., 2:].view(torch.int8).float() * held[..., :2].view(torch.float16).float()
            k, v = held.permute(1, 2, 0, 3, 4, 5).reshape(2, N_HEAD_KV, -1, HEAD_DIM)[:, :, :n]
            score = torch.einsum("thgd,hpd->htgp", q[lo:hi], k) * scale
            seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - (hi - lo), n, device="cuda")[:, None]
            score = torch.where(seen[:, None], score, -math.inf)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            s["out"][layer, lo:hi] = torch.einsum("htgp,hpd->thgd", p, v).reshape(hi - lo, N_HEAD, HEAD_DIM)
    return [s["out"], *_parts(s["pool"])]


def _run_copy(s):
    if own:
        _ok(_bb().pages_copy(s["pool"], s["pool"][0].numel(), s["pages"], s["src_host"], s["dst_host"], s["moved"]))
    else:
        s["pool"][s["dst"]] = s["pool"][s["src"]]
    return s["pool"]


def _run_delta(s):
    if own:
        _ok(_bb().gdn_seqs(s["state"], s["q"], s["k"], s["v"], s["g"], s["beta"], s["out"], s["start"], None, s["workspace"],
                           s["workspace"].numel(), len(s["starts"]) - 1, len(s["starts"]) - 1, s["out"].shape[0], GDN_K_HEADS, GDN_V_HEADS, GDN_DIM, GDN_DIM))
        return [s["out"], s["state"]]
    for i in range(len(s["starts"]) - 1):
        lo, hi = s["starts"][i:i + 2]
        if hi > lo:
            _plain_delta(*(s[x][lo:hi] for x in ("q", "k", "v", "g", "beta", "out")), s["state"][i])
    return [s["out"], s["state"]]


def _plain_delta(q, k, v, g, beta, out, state):
    """One sequence, in chunks of 64 tokens.  With G the sums of g since the chunk's begin, the updates u of a chunk solve
    u_i = beta_i (v_i - e^G_i k_i S) - sum over j < i of beta_i e^(G_i - G_j) (k_i . k_j) u_j."""
    n, c = q.shape[0], min(64, q.shape[0])
    m = -(-n // c)
    chunked = lambda x: torch.cat([x, x.new_zeros(m * c - n, *x.shape[1:])]).reshape(m, c, *x.shape[1:]).transpose(1, 2)  # noqa: E731
    heads = lambda x: chunked(x).repeat_interleave(GDN_V_HEADS // GDN_K_HEADS, 1)  # noqa: E731
    q, k, v, g, beta = heads(q), heads(k), chunked(v), chunked(g).double().cumsum(-1), chunked(beta)      # [chunks, heads, c, ...]
    low = torch.ones(c, c, dtype=torch.bool, device="cuda").tril()
    decay = torch.where(low, (g[..., :, None] - g[..., None, :]).exp(), 0.0).float()
    a = torch.where(low.tril(-1), beta[..., None] * decay * (k @ k.mT), 0.0)
    # rows of the inverse of 1 + a, one after the other, for all chunks at once
    inv = torch.eye(c, device="cuda").expand_as(a).clone()
    for i in range(1, c):
        inv[..., i, :i] = -(a[..., i, None, :i] @ inv[..., :i, :i])[..., 0, :]
    inv = inv * beta[..., None, :]
    weight = decay * (q @ k.mT)
    since, left, last = g.exp().float()[..., None], (g[..., -1:] - g).exp().float()[..., None], g[..., -1].exp().float()[..., None, None]
    o = torch.empty_like(v)
    for i in range(m):
        u = inv[i] @ (v[i] - since[i] * (k[i] @ state))
        o[i] = since[i] * (q[i] @ state) + weight[i] @ u
        state.mul_(last[i]).add_(k[i].mT @ (left[i] * u))
    out.copy_(o.transpose(1, 2).reshape(m * c, *out.shape[1:])[:n])


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    """Every input read once, every output written once; two operations per product.  A cache's pages are read where a new
    token sees them."""
    op = case["op"]
    if op == "qk":
        n = case["n_tok"]
        return {"bytes": n * (N_HEAD + N_HEAD_KV) * HEAD_DIM * 8 + 4 * n + 8 * HEAD_DIM, "flops": n * (N_HEAD + N_HEAD_KV) * (4 * HEAD_DIM + 3 * N_ROT)}
    if op == "copy":
        return {"bytes": 2 * case["moved"] * KV_LAYERS * 2 * N_HEAD_KV * PAGE * BLOCKS * BLOCK, "flops": 0}
    new = _ints(case["new"])
    if op == "attend":
        row, n = BLOCKS * BLOCK, sum(new)
        seen = [(c + m, m * c + m * (m + 1) // 2) for c, m in zip(_ints(case["cached"]), new) if m]
        return {"bytes": case["layers"] * (2 * N_HEAD_KV * row * sum(p for p, _ in seen) + n * 4 * HEAD_DIM * (2 * N_HEAD + 2 * N_HEAD_KV)),
                "flops": case["layers"] * 4 * HEAD_DIM * N_HEAD * sum(p for _, p in seen)}
    n, d = sum(new), GDN_DIM
    return {"bytes": 4 * (n * (2 * GDN_K_HEADS * d + 2 * GDN_V_HEADS * d + 2 * GDN_V_HEADS) + sum(1 for m in new if m) * 2 * GDN_V_HEADS * d * d),
            "flops": n * GDN_V_HEADS * 7 * d * d}


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "copy":
        return None
    if op == "qk":
        def head(x, w):
            x = x.double()
            x = w.double() * x * ((x ** 2).sum(-1, keepdim=True) / HEAD_DIM + EPS) ** -0.5
            z = torch.complex(x[..., :N_ROT // 2], x[..., N_ROT // 2:N_ROT])
            z = z * torch.polar(torch.ones_like(s["freq"]), s["pos"].double()[:, None] * s["freq"])[:, None]
            return torch.cat([z.real, z.imag, x[..., N_ROT:]], -1)
        return [head(s["proj"][:, :, :HEAD_DIM], s["q_weight"]), head(s["k"], s["k_weight"])]
    if op == "delta":
        # token by token, all sequences side by side
        out, state = torch.zeros_like(s["out"], dtype=torch.float64), s["state"].double()
        new = _ints(case["new"])
        share = GDN_V_HEADS // GDN_K_HEADS
        for t in range(max(new)):
            who = torch.tensor([i for i, n in enumerate(new) if t < n], device="cuda")
            row = s["start"].long()[who] + t
            q, k = (s[x][row].double().repeat_interleave(share, 1) for x in "qk")
            was = s["g"][row].double().exp()[..., None, None] * state[who]
            miss = s["v"][row].double() - torch.einsum("shk,shkv->shv", k, was)
            state[who] = was + torch.einsum("shk,shv,sh->shkv", k, miss, s["beta"][row].double())
            out[row] = torch.einsum("shk,shkv->shv", q, state[who])
        return [out, state]
    # attention: the cache's rows and the new ones by their bytes, which are defined in fp32; products and softmax in 64 bits
    out = torch.empty_like(s["out"], dtype=torch.float64)
    number = lambda rows: (rows[..., 2:].view(torch.int8).double() * rows[..., :2].view(torch.float16).double()).flatten(-2)  # noqa: E731
    for layer in range(case["layers"]):
        q, fresh = number(_blocks(s["q"][layer])), [number(_blocks(s[x][layer])) for x in "kv"]
        for i, (c, n) in enumerate(zip(_ints(case["cached"]), _ints(case["new"]))):
            lo = s["starts"][i]
            for h in range(N_HEAD if n else 0):
                k, v = (torch.cat([number(s["pool"][s["table"][i].long(), layer, j, h // GROUP]).flatten(0, 1)[:c], fresh[j][lo:lo + n, h // GROUP]])
                        for j in range(2))
                score = q[lo:lo + n, h] @ k.T / math.sqrt(HEAD_DIM)
                score.masked_fill_(torch.ones_like(score, dtype=torch.bool).triu(c + 1), -math.inf)
                out[layer, lo:lo + n, h] = torch.softmax(score, -1) @ v
    return [out, None, None]
