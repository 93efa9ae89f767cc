"""Speculative decoding and weight-based eviction over the 3-bit KV cache: inputs, plain forms and calls.

Four operators of the serving path, on the ring and the paged cache:

* ``tree``: attention of a tree of drafted tokens over the cache.  The drafts are the last positions
  of the cache; each sees every earlier position and the drafts that its bit mask names.
* ``weights``: single-token attention that also adds, for each position and kv head, the attention
  weight that the position received from the query heads of its group.
* ``evict``: the cache is one chunk over its budget; of every (sequence, kv head) the most recent
  positions and the heaviest of the others stay, in order.
* ``commit``: drafted positions are appended, the accepted path of them is kept and the rest dropped.

The cache is given in its stored form: per vector of 128 values 48 bytes of 3-bit codes (least
significant bit first) and (min, max); value = min + code * (max - min) / 7.
"""
import math
import random

import torch

own = False

D = 128
CODE_BYTES = 48
VECTOR_BYTES = 2 * (CODE_BYTES + 8)  # K and V: codes, min and max
T_CLIP = 2.5  # mode T: codes are uniform on [-2.5, 2.5] of the rotated unit vector


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # one user, a short conversation, a small tree: latency
        {"name": "tree short fp32", "op": "tree", "cache": "ring", "mode": "R", "dtype": "float32", "batch": 1,
         "len": 517, "ragged": 0, "draft": 5, "q_heads": 8, "kv_heads": 2},
        # one user, a document in the cache
        {"name": "tree document bf16", "op": "tree", "cache": "ring", "mode": "R", "dtype": "bfloat16", "batch": 1,
         "len": 32768, "ragged": 0, "draft": 16, "q_heads": 32, "kv_heads": 8},
        # a paged batch of unequal requests, rotated codebook
        {"name": "tree paged mode T fp32", "op": "tree", "cache": "paged", "mode": "T", "dtype": "float32",
         "batch": 6, "len": 8191, "ragged": 1237, "draft": 24, "q_heads": 16, "kv_heads": 4},
        # a full server: wide trees over long contexts
        {"name": "tree wide bf16", "op": "tree", "cache": "ring", "mode": "R", "dtype": "bfloat16", "batch": 8,
         "len": 32768, "ragged": 0, "draft": 64, "q_heads": 32, "kv_heads": 8},
        # one user's decode step
        {"name": "weights short", "op": "weights", "batch": 1, "len": 700, "q_heads": 8, "kv_heads": 2},
        {"name": "weights batch 4", "op": "weights", "batch": 4, "len": 8190, "q_heads": 32, "kv_heads": 8},
        # the decode step of the cache's own benchmark
        {"name": "weights batch 32", "op": "weights", "batch": 32, "len": 32768, "q_heads": 32, "kv_heads": 8},
        # budgets of 1k, 8k and 16k positions, evicted a chunk at a time
        {"name": "evict 1k", "op": "evict", "batch": 1, "len": 1088, "keep": 1001, "recent": 128, "kv_heads": 2},
        {"name": "evict 8k", "op": "evict", "batch": 4, "len": 8704, "keep": 8192, "recent": 1024, "kv_heads": 8},
        {"name": "evict 16k", "op": "evict", "batch": 16, "len": 17408, "keep": 16384, "recent": 2048,
         "kv_heads": 8},
        # after a verification step: a chain of a small tree, and of a batch of wide ones
        {"name": "commit 1", "op": "commit", "batch": 1, "len": 2000, "draft": 8, "accepted": 3, "kv_heads": 8},
        {"name": "commit 32", "op": "commit", "batch": 32, "len": 4097, "draft": 64, "accepted": 9, "kv_heads": 8},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "weights", "evict", "commit"])
    kv = rng.choice([1, 2, 3, 4, 8])
    if op == "tree":
        group, draft = rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), _log_int(rng, 1, 64)
        batch = _log_int(rng, 1, 16)
        most = min(40000, 8 * 64 * 32 * 32768 // (batch * draft * group * kv), 8 * 8 * 32768 // (batch * kv))
        length = _log_int(rng, draft, max(draft, most))
        ragged = rng.choice([0, rng.randint(1, max(1, length // batch))])
        cache = "paged" if ragged else rng.choice(["ring", "paged"])
        return {"op": op, "cache": cache, "mode": rng.choice(["R", "R", "T"]),
                "dtype": rng.choice(["float32", "bfloat16"]), "batch": batch, "len": length, "ragged": ragged,
                "draft": draft, "q_heads": group * kv, "kv_heads": kv}
    if op == "weights":
        group, batch = rng.choice([1, 2, 3, 4, 5, 7, 8]), _log_int(rng, 1, 32)
        return {"op": op, "batch": batch, "len": _log_int(rng, 1, min(40000, 32 * 32768 * 8 // (batch * kv * 2))),
                "q_heads": group * kv, "kv_heads": kv}
    if op == "evict":
        batch = _log_int(rng, 1, 16)
        keep = _log_int(rng, 1, min(40000, 16 * 16384 * 8 // (batch * kv)))
        length = keep + _log_int(rng, 1, max(1, min(keep, 1024)))
        return {"op": op, "batch": batch, "len": length, "keep": keep, "recent": rng.randint(0, keep),
                "kv_heads": kv}
    draft = rng.randint(1, 64)
    return {"op": op, "batch": _log_int(rng, 1, 32), "len": _log_int(rng, 1, 8192) + draft, "draft": draft,
            "accepted": rng.randint(1, draft), "kv_heads": kv}


def _lengths(case):
    """Positions of each sequence, drafts included."""
    return [max(case["draft"], case["len"] - b * case["ragged"]) for b in range(case["batch"])]


def work(case):
    B, H = case["batch"], case["kv_heads"]
    if case["op"] == "tree":
        size = 4 if case["dtype"] == "float32" else 2
        rows, positions = B * case["draft"] * case["q_heads"], sum(_lengths(case))
        return {"bytes": positions * H * VECTOR_BYTES + 2 * rows * D * size + 8 * B * case["draft"],
                "flops": 4 * positions * case["draft"] * case["q_heads"] * D}
    if case["op"] == "weights":
        positions = B * case["len"] * H
        return {"bytes": positions * (VECTOR_BYTES + 8) + 2 * B * case["q_heads"] * D * 4,
                "flops": 4 * B * case["len"] * case["q_heads"] * D}
    kept = B * H * (case["keep"] if case["op"] == "evict" else case["accepted"])
    if case["op"] == "evict":
        new = B * H * (case["len"] - case["keep"])
        # the appended chunk in and out, the weights in, indices and weights out, the kept records
        # moved (in and out) and read back (in and out)
        return {"bytes": new * VECTOR_BYTES * 2 + B * H * case["len"] * 8 + kept * (4 + VECTOR_BYTES * 4),
                "flops": 0}
    new = B * H * case["draft"]
    return {"bytes": new * VECTOR_BYTES * 2 + kept * VECTOR_BYTES * 4, "flops": 0}


# ------------------------------------------------------------------ inputs --
def _signs(seed):
    """The 128 signs of mode T's rotation: bit 63 of SplitMix64's draws."""
    out, z, m = [], seed, (1 << 64) - 1
    for _ in range(D):
        z = (z + 0x9E3779B97F4A7C15) & m
        r = z
        r = ((r ^ (r >> 30)) * 0xBF58476D1CE4E5B9) & m
        r = ((r ^ (r >> 27)) * 0x94D049BB133111EB) & m
        r ^= r >> 31
        out.append(-1.0 if r >> 63 else 1.0)
    return out


def _hadamard(dtype):
    h = torch.ones((1, 1), dtype=dtype, device="cuda")
    while h.shape[0] < D:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h


def _store(x, mode, rotation):
    """Stored form of vectors [..., 128]: codes [..., 48] uint8 and (min, max) [..., 2]."""
    if mode == "T":
        norm = x.norm(dim=-1, keepdim=True)
        y = (x / norm) @ rotation
        code = torch.floor((y / T_CLIP + 1) * 4).clamp_(0, 7)
        top = norm * (T_CLIP * 7 / 8 / math.sqrt(D))
        mm = torch.cat([-top, top], -1)
    else:
        lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
        code = torch.round((x - lo) * (7 / (hi - lo))).clamp_(0, 7)
        mm = torch.cat([lo, hi], -1)
    c = code.to(torch.int32).reshape(*x.shape[:-1], 16, 8)
    bits = (c << (3 * torch.arange(8, device=x.device, dtype=torch.int32))).sum(-1, dtype=torch.int32)
    packed = torch.stack([bits & 255, (bits >> 8) & 255, (bits >> 16) & 255], -1).to(torch.uint8)
    return packed.reshape(*x.shape[:-1], CODE_BYTES), mm.contiguous()


def _vectors(gen, batch, n, heads, mode, rotation, spread):
    """Stored K or V of `batch` sequences: channels of unequal spread, as projections have them."""
    codes, mms = [], []
    step = max(1, (1 << 20) // (n * heads))
    for b in range(0, batch, step):
        k = min(step, batch - b)
        x = torch.randn((k, n, heads, D), generator=gen, device="cuda") * spread
        c, m = _store(x, mode, rotation)
        codes.append(c)
        mms.append(m)
    return torch.cat(codes), torch.cat(mms)


def _tree(r, draft):
    """Ancestor masks of a random tree (a draft sees itself and its ancestors), as signed 64-bit words."""
    masks = []
    for i in range(draft):
        parent = r.randint(max(-1, i - 5), i - 1) if i else -1
        masks.append((1 << i) | (masks[parent] if parent >= 0 else 0))
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def _chain(r, draft, accepted):
    """Offsets of an accepted path within the drafts, ascending."""
    return sorted(r.sample(range(draft), accepted))


def prepare(case, seed):
    r = random.Random(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    B, H, n = case["batch"], case["kv_heads"], case["len"]
    mode = case.get("mode", "R")
    s = {"case": dict(case), "signs": None, "rotation": None}
    if mode == "T":
        s["signs"] = torch.tensor(_signs(seed), device="cuda")
        s["rotation"] = s["signs"][:, None] * _hadamard(torch.float32)  # y = v @ rotation
    spread = 0.5 + torch.rand((H, D), generator=gen, device="cuda")
    for name in ("k", "v"):
        s[name], s[name + "mm"] = _vectors(gen, B, n, H, mode, s["rotation"], spread)
    if case["op"] == "tree":
        T, dtype = case["draft"], getattr(torch, case["dtype"])
        s["q"] = (2 * torch.randn((B, T, case["q_heads"], D), generator=gen, device="cuda")).to(dtype)
        s["mask"] = torch.tensor([_tree(r, T) for _ in range(B)], dtype=torch.int64, device="cuda")
        s["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    elif case["op"] == "weights":
        s["q"] = 2 * torch.randn((B, case["q_heads"], D), generator=gen, device="cuda")
        # what the positions received in the last few steps
        s["weights"] = torch.rand((B, H, n + 37), generator=gen, device="cuda") * (8 * case["q_heads"] / H / n)
    elif case["op"] == "evict":
        w = torch.exp(3 * torch.randn((B, H, n), generator=gen, device="cuda"))
        s["weights"] = torch.where(torch.rand(w.shape, generator=gen, device="cuda") < 0.05, torch.zeros_like(w), w)
    else:
        s["path"] = torch.tensor([_chain(r, case["draft"], case["accepted"]) for _ in range(B)], dtype=torch.int32,
                                 device="cuda") + (n - case["draft"])
    # positions that a pass appends: the chunk over the budget, or the drafts
    held = case["keep"] if case["op"] == "evict" else n - case["draft"] if case["op"] == "commit" else n
    s["held"] = held
    s["new"] = [s[x][:, held:].clone() for x in ("k", "kmm", "v", "vmm")]
    if own:
        s["cache"] = _cache(case, s, seed)
    return s


def _cache(case, s, seed):
    """The framework's cache that holds the prepared positions."""
    from ferrisres_b200 import kv, paged
    stored = [s[x].reshape(case["batch"], case["len"], -1) if x in ("k", "v") else s[x]
              for x in ("k", "kmm", "v", "vmm")]
    mode = case.get("mode", "R")
    if case.get("cache") == "paged":
        lens = _lengths(case)
        c = paged.PagedKv3Cache(1, sum(-(-x // 32) for x in lens) + 1, case["kv_heads"], mode=mode, seed=seed)
        s["requests"] = [c.create_request() for _ in lens]
        for b, x in enumerate(lens):
            c.append_packed(0, [s["requests"][b]], *[t[b:b + 1, :x] for t in stored])
        return c
    c = kv.Kv3Cache(case["batch"], case["kv_heads"], case["len"] + 64, mode=mode, seed=seed)
    if s["held"]:
        c.append_packed(*[t[:, :s["held"]].contiguous() for t in stored])
    return c


# -------------------------------------------------------------- plain forms --
def _load(codes, mm, rotation):
    """Values [B, H, n, 128] of stored vectors [B, n, H, .]."""
    b = codes.reshape(*codes.shape[:-1], 16, 3).to(torch.int32)
    bits = b[..., 0] | (b[..., 1] << 8) | (b[..., 2] << 16)
    shift = 3 * torch.arange(8, device=codes.device, dtype=torch.int32)
    c = ((bits[..., None] >> shift) & 7).reshape(*codes.shape[:-1], D).to(torch.float32)
    x = mm[..., :1] + c * ((mm[..., 1:] - mm[..., :1]) / 7)
    if rotation is not None:  # back through the orthogonal rotation
        x = (x @ rotation.t()) / math.sqrt(D)
    return x.transpose(1, 2)


def _softmax(x):
    """Row softmax in 32 bits; a row that sees nothing gets weights of 0."""
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _tree_plain(s):
    q, (B, T, Hq, _) = s["q"], s["q"].shape
    H, n = s["case"]["kv_heads"], s["case"]["len"]
    G = Hq // H
    k, v = _load(s["k"], s["kmm"], s["rotation"]), _load(s["v"], s["vmm"], s["rotation"])
    rows = q.float().reshape(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D)
    x = (rows @ k.transpose(2, 3)) / math.sqrt(D)
    # draft j of sequence b is position lens[b] - T + j
    at = torch.arange(n, device=q.device)[None, :] - (s["lens"][:, None] - T)
    bit = (s["mask"][:, :, None] >> at.clamp(0, T - 1)[:, None, :]) & 1
    sees = (at < 0)[:, None, :] | ((at < T)[:, None, :] & (bit == 1))
    sees = sees[:, None, :, None, :].expand(B, 1, T, G, n).reshape(B, 1, T * G, n)
    p = _softmax(x.masked_fill_(~sees, -math.inf))
    out = (p @ v).reshape(B, H, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, Hq, D)
    return out.to(q.dtype)


def _weights_plain(s):
    q, (B, Hq, _) = s["q"], s["q"].shape
    H, n = s["case"]["kv_heads"], s["case"]["len"]
    k, v = _load(s["k"], s["kmm"], None), _load(s["v"], s["vmm"], None)
    p = _softmax((q.reshape(B, H, Hq // H, D) @ k.transpose(2, 3)) / math.sqrt(D))
    s["weights"][:, :, :n] += p.sum(2)
    return {"out": (p @ v).reshape(B, Hq, D), "weights": s["weights"]}


def _append_plain(s):
    for name, new in zip(("k", "kmm", "v", "vmm"), s["new"]):
        s[name][:, s["held"]:] = new


def _evict_plain(s):
    case, w = s["case"], s["weights"]
    n, keep, recent = case["len"], case["keep"], case["recent"]
    _append_plain(s)
    order = torch.sort(w[:, :, :n - recent], dim=-1, descending=True, stable=True).indices
    heavy = torch.sort(order[:, :, :keep - recent], dim=-1).values
    last = torch.arange(n - recent, n, device=w.device).expand(*w.shape[:2], recent)
    index = torch.cat([heavy, last], -1)
    at = index.transpose(1, 2)[..., None]
    for name in ("k", "kmm", "v", "vmm"):
        s[name][:, :keep] = torch.gather(s[name], 1, at.expand(*at.shape[:3], s[name].shape[-1]))
    weights = torch.zeros_like(w)
    weights[:, :, :keep] = torch.gather(w, 2, index)
    return {"index": index.to(torch.int32), "weights": weights, "cache": _stored_plain(s, 0, keep)}


def _stored_plain(s, start, end):
    B = s["case"]["batch"]
    return [s[x][:, start:end].reshape(B, end - start, -1) if x in ("k", "v") else s[x][:, start:end]
            for x in ("k", "kmm", "v", "vmm")]


def _commit_plain(s):
    _append_plain(s)
    at, start = s["path"].long()[:, :, None, None], s["held"]
    end = start + s["case"]["accepted"]
    for name in ("k", "kmm", "v", "vmm"):
        s[name][:, start:end] = torch.gather(s[name], 1, at.expand(-1, -1, *s[name].shape[2:]))
    return _stored_plain(s, start, end)


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        plain = {"tree": _tree_plain, "weights": _weights_plain, "evict": _evict_plain, "commit": _commit_plain}
        return plain[op](s)
    c, case = s["cache"], s["case"]
    if op == "tree":
        if case["cache"] == "paged":
            return c.tree_decode(0, s["requests"], s["q"], s["mask"])
        return c.tree_decode(s["q"], s["mask"])
    if op == "weights":
        return {"out": c.flash_decode(s["q"], weights=s["weights"]), "weights": s["weights"]}
    k, kmm, v, vmm = s["new"]
    c.append_packed(k.flatten(2), kmm, v.flatten(2), vmm)
    if op == "evict":
        index, weights = c.evict_heavy(s["weights"], case["keep"], case["recent"])
        return {"index": index, "weights": weights, "cache": list(c.export_range(0, case["keep"]))}
    # the path is kept, and the oldest positions make room: the cache stays as long as it was
    c.keep(s["path"], start=s["held"])
    out = list(c.export_range(s["held"], s["held"] + case["accepted"]))
    c.evict_front(case["accepted"])
    return out


# --------------------------------------------------------- from the definition --
def exact(case, seed):
    """Attention outputs in 64 bits, one kv head at a time; the other operators only move and choose."""
    if case["op"] not in ("tree", "weights"):
        return None
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    B, H, n, Hq = case["batch"], case["kv_heads"], case["len"], case["q_heads"]
    G = Hq // H
    tree = case["op"] == "tree"
    q = s["q"].double() if tree else s["q"].double()[:, None]
    T = q.shape[1]
    lens = _lengths(case) if tree else [n] * B
    out = torch.zeros((B, T, Hq, D), dtype=torch.float64, device="cuda")
    weights = None if tree else s["weights"].double()
    place = torch.arange(D, device="cuda") * 3
    undo = None
    if case.get("mode") == "T":
        undo = _hadamard(torch.float64) * torch.tensor(_signs(seed), dtype=torch.float64, device="cuda") / math.sqrt(D)

    def values(codes, mm):
        wide = torch.nn.functional.pad(codes.to(torch.int64), (0, 1))  # a code may straddle two bytes
        two = wide[:, place // 8] + 256 * wide[:, place // 8 + 1]
        c = torch.bitwise_and(torch.bitwise_right_shift(two, place % 8), 7).double()
        lo, hi = mm[:, :1].double(), mm[:, 1:].double()
        x = lo + c * (hi - lo) / 7
        return x if undo is None else x @ undo

    for b in range(B):
        n_b = lens[b]
        allowed = torch.ones((T, n_b), dtype=torch.bool, device="cuda")
        if tree:
            allowed[:, n_b - T:] = torch.tensor(
                [[bool((m >> j) & 1) for j in range(T)] for m in s["mask"][b].tolist()], device="cuda")
        for h in range(H):
            k = values(s["k"][b, :n_b, h], s["kmm"][b, :n_b, h])
            v = values(s["v"][b, :n_b, h], s["vmm"][b, :n_b, h])
            for g in range(h * G, h * G + G):
                x = torch.where(allowed, q[b, :, g] @ k.T / D ** 0.5, -math.inf)
                p = torch.softmax(x, -1)
                out[b, :, g] = p @ v
                if weights is not None:
                    weights[b, h, :n_b] += p[0]
    return out if tree else {"out": out[:, 0], "weights": weights}
