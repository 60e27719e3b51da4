"""The 8-bit key/value cache's operators as a user's program calls them, with their plain forms.

Three operators over a cache that holds keys and values in 8 bits, one scale for each block of 32 tokens and
key/value head (K and V apart): appending new rows, attention over the cache, and eviction by accumulated
attention weight.  With X the appended fp32 rows:

    scale  d  = fl32(max |X| over the block's present tokens and channels / 127)
    code   q  = nearest integer to X / d (ties to even);  the cache stands for fl32(q d)
    attention: p = softmax over the permitted keys of (q_row . K') / sqrt(D);  out = p V'
    weight of a key: the sum of its p over the sequence's query rows and the heads that share its kv head
    eviction: per (sequence, kv head) the last `recent` tokens and the heaviest of the others, in their order

The plain forms are vectorised over sequences padded to the longest one.
"""
import math

import torch

own = False

BLOCK = 32


# ------------------------------------------------------------------- cases ---

def listed():
    return [
        # one new token for each of eight chats: the append of a decode step, where launch latency counts
        dict(name="append-token-8", op="append", seqs=8, kv=4, dim=128, cap=777, rows=1, ragged=True),
        # a whole prompt into an empty cache
        dict(name="append-prompt-4096", op="append", seqs=1, kv=4, dim=128, cap=4096, rows=4096, ragged=False),
        # chunks of prompts of different lengths, as many kv heads as a vision encoder has
        dict(name="append-chunks-5", op="append", seqs=5, kv=16, dim=80, cap=2900, rows=1001, ragged=True),
        # the smallest decode step: one chat, one token
        dict(name="decode-1x1000", op="attend", seqs=1, heads=28, kv=4, dim=128, cap=1000, rows=1, ragged=False, causal=True, weights=False),
        # a decode step of eight chats at the VL decoder's head layout
        dict(name="decode-8x4096", op="attend", seqs=8, heads=28, kv=4, dim=128, cap=4096, rows=1, ragged=True, causal=True, weights=False),
        # a decode step over long documents: bound by reading the cache
        dict(name="decode-8x65536", op="attend", seqs=8, heads=28, kv=4, dim=128, cap=65536, rows=1, ragged=True, causal=True, weights=False),
        # a decode step that also keeps the running weights which eviction goes by; every head has its own keys
        dict(name="decode-weights-6x3001", op="attend", seqs=6, heads=16, kv=16, dim=64, cap=3001, rows=1, ragged=True, causal=True, weights=True),
        # eight rows of one chat at a time (a short turn, or drafts to verify)
        dict(name="rows8-1x4096", op="attend", seqs=1, heads=28, kv=4, dim=128, cap=4096, rows=8, ragged=False, causal=True, weights=False),
        # a whole prompt against itself
        dict(name="prompt-4096", op="attend", seqs=1, heads=28, kv=4, dim=128, cap=4096, rows=4096, ragged=False, causal=True, weights=False),
        # chunks of different lengths over what came before, non-causal, with weights, an odd head size
        dict(name="chunks-weights-5", op="attend", seqs=5, heads=16, kv=16, dim=80, cap=1501, rows=701, ragged=True, causal=False, weights=True),
        # a chat's cache cut to half
        dict(name="evict-2x2048", op="evict", seqs=2, kv=4, dim=128, cap=2048, keep=1024, recent=64, ragged=False),
        # long caches of a batch cut to a quarter
        dict(name="evict-8x32768", op="evict", seqs=8, kv=4, dim=128, cap=32768, keep=8191, recent=255, ragged=True),
    ]


HEADS = [(28, 4, 128), (28, 2, 128), (7, 1, 128), (24, 24, 128), (8, 2, 64), (16, 16, 64), (16, 16, 80), (8, 8, 80)]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    heads, kv, dim = rng.choice(HEADS)
    seqs = rng.choice([1, 1, 2, 3, 5, 8])
    kind = rng.choice(["token", "prompt", "decode", "decode", "rows", "chunks", "chunks", "evict"])
    ragged = seqs > 1
    if kind in ("token", "prompt"):
        rows = 1 if kind == "token" else _log(rng, 2, max(2, 4096 * 512 // (kv * dim * seqs)))
        return dict(op="append", seqs=seqs, kv=kv, dim=dim, cap=rows + _log(rng, 1, 4096), rows=rows, ragged=ragged)
    if kind == "evict":
        cap = _log(rng, 64, max(64, 8 * 32768 * 512 // (kv * dim * seqs) // 2))
        keep = _log(rng, 16, cap - 1)
        return dict(op="evict", seqs=seqs, kv=kv, dim=dim, cap=cap, keep=keep, recent=rng.randint(0, keep), ragged=ragged)
    if kind == "chunks":
        rows = _log(rng, 9, 2048)
        most = 28 * 4096 * 4096 // (heads * seqs * rows)  # the scores of the largest listed prompt
        cap = _log(rng, rows, max(rows, min(8192, most)))
    else:
        rows = 1 if kind == "decode" else rng.randint(2, 8)
        cap = _log(rng, rows, min(65536, 8 * 65536 * 512 // (kv * dim * seqs) // 2))
    return dict(op="attend", seqs=seqs, heads=heads, kv=kv, dim=dim, cap=cap, rows=rows, ragged=ragged,
                causal=rng.random() < 0.75, weights=rng.random() < 0.35)


def _sizes(case):
    """Each sequence's length (with its new rows) and number of new rows."""
    S, cap, rows, ragged = case["seqs"], case["cap"], case.get("rows", 0), case["ragged"]
    new = [max(1, rows - (s * rows * 3) // (4 * S)) if ragged and rows > 1 else rows for s in range(S)]
    lens = [max(n, cap - (s * cap * 5) // (8 * S) - s) if ragged else cap for s, n in enumerate(new)]
    if case["op"] == "append" and rows > 1:
        # chunks start at a block's begin, so that the rewind before each pass gives back exactly what was there
        lens = [(t - n) // BLOCK * BLOCK + n for t, n in zip(lens, new)]
    return lens, new


def work(case):
    lens, new = _sizes(case)
    row = case["kv"] * case["dim"]
    if case["op"] == "append":
        open_rows = sum((t - n) % BLOCK for t, n in zip(lens, new))
        shown = sum((t - n) % BLOCK + n for t, n in zip(lens, new))
        return {"bytes": 2 * row * (4 * (sum(new) + open_rows) + sum(new) + 4 * shown), "flops": 0}
    if case["op"] == "evict":
        kept = sum(min(t, case["keep"]) for t in lens)
        return {"bytes": 4 * sum(lens) * case["kv"] + 2 * row * kept * 6 + 8 * case["kv"] * kept, "flops": 0}
    heads, dim = case["heads"], case["dim"]
    seen = sum(n * t - (n * (n - 1) // 2 if case["causal"] else 0) for t, n in zip(lens, new))
    b = 2 * sum(lens) * row + 8 * sum(-(-t // BLOCK) for t in lens) * case["kv"] + 8 * sum(new) * heads * dim
    return {"bytes": b + (8 * sum(lens) * case["kv"] if case["weights"] else 0), "flops": 4 * heads * dim * seen}


# ------------------------------------------------------------------ inputs ---

def _inputs(case, seed):
    """Rows as a decoder makes them: channels with an offset of their own in K, tokens of different magnitude in both."""
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    r = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    lens, new = _sizes(case)
    S, T, row = case["seqs"], max(lens), case["kv"] * case["dim"]
    x = {"k": (r(S, T, row) + 0.7 * r(row)) * torch.exp(0.3 * r(S, T, 1)), "v": r(S, T, row) * torch.exp(0.5 * r(S, T, 1))}
    if case["op"] == "attend":
        x["q"] = 1.2 * r(sum(new), case["heads"] * case["dim"])
        if case["weights"]:
            x["w"] = 3 * torch.rand((S, case["kv"], case["cap"]), generator=g, device="cuda") ** 6
    if case["op"] == "evict":
        # a few heavy tokens, many light ones, ties among those that nothing looked at
        w = 5 * torch.rand((S, case["kv"], case["cap"]), generator=g, device="cuda") ** 8
        x["w"] = torch.where(w < 1e-9, torch.zeros_like(w), w)
    return x


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    x = _inputs(case, seed)
    lens, new = _sizes(case)
    S, H, D, T = case["seqs"], case["kv"], case["dim"], max(lens)
    before = [t - n for t, n in zip(lens, new)] if case["op"] == "append" else lens  # tokens in the cache before the pass
    starts = _starts(new)
    st = {"op": case["op"], "S": S, "H": H, "D": D, "T": T, "cap": case["cap"]}
    # packed rows: rows [starts[s], starts[s + 1]) are sequence s's
    pack = lambda t, first, count: torch.cat([t[s, a:a + n] for s, (a, n) in enumerate(zip(first, count))])  # noqa: E731
    st["starts"] = _int(starts) if S > 1 else None
    st["nmax"] = max(new)
    if own:
        from pixelina_b200 import pxq

        pxq.init(0)
        cache = pxq.KVCache(S, case["cap"], H, D)
        zero = [0] * S
        if sum(before):
            cache.append(pack(x["k"], zero, before), pack(x["v"], zero, before), starts=_int(_starts(before)))
        st["pxq"], st["cache"] = pxq, cache
    else:
        live = torch.arange(T, device="cuda") < _int(before)[:, None]
        if case["op"] != "append":
            for n in ("k", "v"):
                st[n + "_codes"], st[n + "_scale"] = _quantize(x[n].view(S, T, H, D), live)
    if case["op"] == "append":
        first = [b // BLOCK * BLOCK for b in before]
        st["first"], st["before"] = _int(first), _int(before)
        st["count"] = max(t - f for t, f in zip(lens, first))
        st["k_new"], st["v_new"] = pack(x["k"], before, new), pack(x["v"], before, new)
        if own:
            st["k_out"], st["v_out"] = torch.zeros((2, S, st["count"], H * D), device="cuda")
        else:
            st["k_open"], st["v_open"] = (torch.stack([_pad(x[n][s, f:b], BLOCK) for s, (f, b) in enumerate(zip(first, before))])
                                          for n in ("k", "v"))
            # where each token shown comes from: its sequence's open block, then the new rows; -1: nothing
            at = [[s * BLOCK + i if f + i < b else S * BLOCK + starts[s] + f + i - b if f + i < t else -1
                   for i in range(-(-st["count"] // BLOCK) * BLOCK)] for s, (f, b, t) in enumerate(zip(first, before, lens))]
            st["at"] = torch.tensor(at, device="cuda")
    if case["op"] == "attend":
        st["q"], st["heads"], st["causal"] = x["q"], case["heads"], case["causal"]
        st["weights"] = x.get("w")
        st["weights_out"] = torch.zeros_like(x["w"]) if case["weights"] else None
        if not own:
            n, t = _int(new)[:, None], _int(lens)[:, None]
            i = torch.arange(st["nmax"], device="cuda")[None, :]
            st["row_at"] = torch.where(i < n, _int(starts[:-1])[:, None] + i, 0)
            seen = (t - n + i + 1).clamp(min=0) if case["causal"] else t.expand(S, st["nmax"])
            st["seen"] = torch.where(i < n, seen, 0)
            st["take"] = torch.tensor([s * st["nmax"] + j for s in range(S) for j in range(new[s])], device="cuda")
            st["lens"] = _int(lens)
    if case["op"] == "evict":
        st["w"], st["keep"], st["recent"] = x["w"], case["keep"], case["recent"]
        if own:
            st["dst"] = pxq.KVCache(S, case["keep"], H, D)
            st["k_out"], st["v_out"] = torch.zeros((2, S, case["keep"], H * D), device="cuda")
            st["w_out"] = torch.zeros((S, H, case["keep"]), device="cuda")
            st["kept"] = torch.full((S, H, case["keep"]), -1, dtype=torch.int32, device="cuda")
        else:
            st["lens"] = _int(lens)
    return st


def _pad(x, n):
    return torch.cat([x, x.new_zeros((n - x.shape[0],) + x.shape[1:])])


# ------------------------------------------------------------- plain forms ---

def _quantize(x, live):
    """Rows [S, T, H, D] and which of them are present -> codes [S, H, T', D] (int8) and scales [S, H, T' / 32], T' whole blocks."""
    S, T, H, D = x.shape
    nb = -(-T // BLOCK)
    x = torch.nn.functional.pad(x * live[:, :, None, None], (0, 0, 0, 0, 0, nb * BLOCK - T))
    x = x.permute(0, 2, 1, 3).reshape(S, H, nb, BLOCK * D)
    a = x.abs().amax(-1)
    d = torch.where(a < 2.0 ** -118, torch.zeros_like(a), (a.double() / 127).float())
    # the quotient in 64 bits: in 32, values next to a border fall on either side of it
    q = torch.round(x.double() / torch.where(d > 0, d, torch.ones_like(d)).double()[..., None])
    q = torch.where(d[..., None] > 0, q, torch.zeros_like(q)).to(torch.int8)
    return q.view(S, H, nb * BLOCK, D), d


def _values(codes, scale):
    S, H, T, D = codes.shape
    return (codes.view(S, H, T // BLOCK, BLOCK * D).float() * scale[..., None]).view(S, H, T, D)


def _plain_append(st):
    S, H, D, n = st["S"], st["H"], st["D"], st["count"]
    live = st["at"] >= 0

    def one(opened, new):
        rows = torch.cat([opened.reshape(-1, H * D), new])
        x = rows[st["at"].clamp(min=0).reshape(-1)].view(S, -1, H, D)
        shown = _values(*_quantize(x, live))
        return (shown.permute(0, 2, 1, 3) * live[:, :, None, None]).reshape(S, -1, H * D)[:, :n]

    return one(st["k_open"], st["k_new"]), one(st["v_open"], st["v_new"])


def _plain_attend(st):
    S, H, D, heads, n = st["S"], st["H"], st["D"], st["heads"], st["nmax"]
    G = heads // H
    k, v = _values(st["k_codes"], st["k_scale"]), _values(st["v_codes"], st["v_scale"])
    T = k.shape[2]
    q = st["q"][st["row_at"].reshape(-1)].view(S, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(S, H, n * G, D)
    z = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(D))
    hide = torch.arange(T, device=z.device) >= st["seen"][:, :, None]  # [S, n, T]
    z.view(S, H, n, G, T).masked_fill_(hide[:, None, :, None, :], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = z.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    out = (p @ v).view(S, H, n, G, D).permute(0, 2, 1, 3, 4).reshape(S * n, heads * D)[st["take"]]
    if st["weights"] is None:
        return out
    cap = st["cap"]
    w = torch.nn.functional.pad(p.sum(2), (0, max(0, cap - T)))[..., :cap]
    live = torch.arange(cap, device=w.device) < st["lens"][:, None, None]
    return out, torch.where(live, st["weights"] + w, torch.zeros_like(w))


def _plain_evict(st):
    S, H, D, keep = st["S"], st["H"], st["D"], st["keep"]
    lens, w = st["lens"][:, None, None], st["w"]
    j = torch.arange(w.shape[-1], device=w.device)
    key = torch.where(torch.isnan(w), -math.inf, w)
    key = torch.where(j >= lens - st["recent"], math.inf, key)
    key = torch.where(j >= lens, -math.inf, key)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    count = torch.minimum(lens, torch.full_like(lens, keep))
    there = torch.arange(keep, device=w.device) < count
    at = torch.where(there, best, w.shape[-1]).sort(-1).values.clamp(max=w.shape[-1] - 1)  # [S, H, keep]

    def one(codes, scale):
        pick = at[..., None].expand(S, H, keep, D)
        q = torch.gather(codes, 2, pick).float()
        x = q * torch.gather(scale, 2, at // BLOCK)[..., None]
        y = _values(*_quantize(x.permute(0, 2, 1, 3), there[:, 0]))[:, :, :keep]
        return (y * there[..., None]).permute(0, 2, 1, 3).reshape(S, keep, H * D)

    k, v = one(st["k_codes"], st["k_scale"]), one(st["v_codes"], st["v_scale"])
    return k, v, torch.where(there, torch.gather(w, 2, at), 0.0), torch.where(there, at, -1).to(torch.int32)


def run(st):
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[st["op"]](st)
    pxq, cache = st["pxq"], st["cache"]
    if st["op"] == "append":
        cache.truncate(st["before"])
        cache.append(st["k_new"], st["v_new"], starts=st["starts"])
        return cache.read(st["first"], st["count"], k=st["k_out"], v=st["v_out"])
    if st["op"] == "attend":
        out = pxq.kv_attention(st["q"], cache, st["heads"], starts=st["starts"], max_rows=st["nmax"], causal=st["causal"],
                               weights=st["weights"], weights_out=st["weights_out"])
        return out if st["weights"] is None else (out, st["weights_out"])
    pxq.kv_evict(cache, st["dst"], st["w"], recent=st["recent"], weights_out=st["w_out"], kept=st["kept"])
    k, v = st["dst"].read(None, st["keep"], k=st["k_out"], v=st["v_out"])
    return k, v, st["w_out"], st["kept"]


# ------------------------------------------------------------------- exact ---

def _exact_cache(rows):
    """[t, H, D] fp32 rows of one sequence -> the fp32 values that the cache stands for, block by block in 64 bits."""
    t, H, D = rows.shape
    out = torch.empty_like(rows)
    whole = t // BLOCK * BLOCK
    for a, b in ((0, whole), (whole, t)):
        if a == b:
            continue
        x = rows[a:b].double().view(-1, min(BLOCK, b - a), H, D)
        d = (x.abs().amax(dim=(1, 3), keepdim=True) / 127.0).float().double()
        d = torch.where(d * 127 < 2.0 ** -118, torch.ones_like(d), d)
        out[a:b] = (torch.round(x / d) * d).float().view(b - a, H, D)
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    lens, new = _sizes(case)
    S, H, D = case["seqs"], case["kv"], case["dim"]
    if case["op"] == "append":
        first = [(t - n) // BLOCK * BLOCK for t, n in zip(lens, new)]
        count = max(t - f for t, f in zip(lens, first))
        both = []
        for n in ("k", "v"):
            y = torch.zeros((S, count, H * D), dtype=torch.float64, device="cuda")
            for s in range(S):
                y[s, :lens[s] - first[s]] = _exact_cache(x[n][s, first[s]:lens[s]].view(-1, H, D)).reshape(-1, H * D)
            both.append(y)
        return tuple(both)
    if case["op"] == "evict":
        keep, recent = case["keep"], case["recent"]
        k = torch.zeros((S, keep, H, D), dtype=torch.float64, device="cuda")
        v, w = torch.zeros_like(k), torch.zeros((S, H, keep), dtype=torch.float64, device="cuda")
        kept = torch.full((S, H, keep), -1, dtype=torch.int32, device="cuda")
        for s, t in enumerate(lens):
            c = min(t, keep)
            values = [_exact_cache(x[n][s, :t].view(t, H, D)) for n in ("k", "v")]
            for h in range(H):
                old = max(0, t - recent)
                order = torch.argsort(-x["w"][s, h, :old].double(), stable=True)[:max(0, c - (t - old))]
                last = torch.arange(max(old, t - c), t, device="cuda")
                at = torch.cat([order, last]).sort().values
                for y, val in zip((k, v), values):
                    y[s, :c, h] = _exact_cache(val[at, h][:, None]).double()[:, 0]
                w[s, h, :c] = x["w"][s, h, at].double()
                kept[s, h, :c] = at.int()
        return k.view(S, keep, H * D), v.view(S, keep, H * D), w, kept
    heads, causal = case["heads"], case["causal"]
    G, at = heads // H, _starts(new)
    out = torch.empty((sum(new), heads, D), dtype=torch.float64, device="cuda")
    w = torch.zeros((S, H, case["cap"]), dtype=torch.float64, device="cuda")
    for s, (t, n) in enumerate(zip(lens, new)):
        k, v = (_exact_cache(x[m][s, :t].view(t, H, D)).double() for m in ("k", "v"))
        q = x["q"][at[s]:at[s + 1]].double().view(n, heads, D)
        hide = torch.ones((n, t), dtype=torch.bool, device="cuda").triu(t - n + 1) if causal else None
        for h in range(heads):
            z = q[:, h] @ k[:, h // G].T / math.sqrt(D)
            if hide is not None:
                z.masked_fill_(hide, -math.inf)
            p = torch.softmax(z, -1)
            out[at[s]:at[s + 1], h] = p @ v[:, h // G]
            if case["weights"]:
                w[s, h // G, :t] += p.sum(0)
        if case["weights"]:
            w[s, :, :t] += x["w"][s, :, :t].double()
    out = out.view(sum(new), heads * D)
    return (out, w) if case["weights"] else out
