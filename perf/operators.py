"""The work that the paged-cache operators are measured on: attention of one new token a sequence over a paged key / value
cache, rows written into its pages, block tables and slot maps built from request lengths, and pages given back.

`own` false: each operator in its plain form, elementary torch operations in 32 bits (integers in 64).  True: the public entry
points, called as a serving loop calls them.

A case is a dict of plain values.  Common to all:
  op        "attend", "write", "extend" or "release"
  page      tokens in a page of the cache
Attention and rows:
  H, Hkv, D query heads, key / value heads, head dimension;  dtype  "bf16" or "fp16"
Attention:
  B         sequences, of which the last `idle` have no token (rows that pad a batch to a captured size)
  shortest, longest   their lengths, spread over this range
  bias      "none", "float" (B, H, N) in q's dtype, "f32" (H, N) in fp32 expanded over the batch (a table by position),
            "mask" (B, N) bool expanded over the heads
Rows:
  T         tokens, of which every `skip`-th has no slot (0: all have one);  packed  k and v are slices of one projection
Tables:
  B         requests, holding shortest .. longest tokens each
  new       the most new tokens of a request (1: a decode step; else they are spread over 1 .. new)
  done      every done-th request is finished (release)
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _attend(B, H, Hkv, D, page, shortest, longest, dtype="bf16", bias="none", idle=0):
    return dict(op="attend", B=B, H=H, Hkv=Hkv, D=D, page=page, shortest=shortest, longest=longest, dtype=dtype, bias=bias,
                idle=idle)


def _write(T, Hkv, D, page, dtype="bf16", skip=0, packed=False, G=4):
    return dict(op="write", T=T, Hkv=Hkv, D=D, H=Hkv * G, page=page, dtype=dtype, skip=skip, packed=packed)


def _extend(B, page, shortest, longest, new):
    return dict(op="extend", B=B, page=page, shortest=shortest, longest=longest, new=new)


def _release(B, page, shortest, longest, done):
    return dict(op="release", B=B, page=page, shortest=shortest, longest=longest, done=done)


def listed():
    cases = {
        # the first tokens of a single chat: launches and dependent loads are all there is
        "attend_first_tokens": _attend(1, 32, 8, 128, 16, 17, 17),
        # one long document, odd length, grouped heads: few heads over many keys
        "attend_long": _attend(1, 32, 8, 128, 16, 20011, 20011),
        # a serving batch of chats of very different lengths, rows padded to the captured batch size
        "attend_batch": _attend(64, 32, 8, 128, 16, 200, 8192, idle=3),
        # an encoder-decoder or small model: a key head for each query head, head dimension 64
        "attend_small_heads": _attend(32, 12, 12, 64, 64, 33, 1000, "fp16"),
        # a trained bias a head and position next to grouped heads
        "attend_bias": _attend(8, 32, 4, 128, 32, 2048, 4096, bias="float"),
        # the widest heads, many queries a key head, a padding mask, pages that end inside every tile
        "attend_wide_mask": _attend(16, 32, 2, 256, 24, 100, 4001, bias="mask"),
        # a decode step's new rows, some of them padding
        "write_step": _write(64, 8, 128, 16, skip=9),
        # the prompts of a prefill, sliced out of the fused projection
        "write_prompts": _write(16384, 8, 128, 16, packed=True),
        # a decode step: one token more for each request, some need a page
        "extend_step": _extend(256, 16, 1, 4096, 1),
        # a prefill: many prompts of different lengths, some behind a cached prefix
        "extend_prompts": _extend(64, 16, 0, 512, 4096),
        # a few requests end
        "release_few": _release(256, 16, 1, 4096, 37),
        # a burst of long requests ends
        "release_burst": _release(512, 16, 64, 16384, 2),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(("attend", "attend", "attend", "write", "extend", "release"))
        page = rng.choice((8, 16, 16, 16, 32, 64, 128, 12, 20, 1 if op == "attend" else 48))
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        if op == "attend":
            Hkv, G = rng.choice((1, 2, 3, 4, 6, 8, 8, 16)), rng.choice((1, 2, 3, 4, 4, 5, 7, 8, 8, 12, 16, 32))
            longest = _log_int(rng, 1, 65536)
            c = _attend(_log_int(rng, 1, 256), Hkv * G, Hkv, rng.choice((32, 64, 128, 128, 128, 256)), page,
                        rng.choice((longest, rng.randint(0, longest))), longest, dtype,
                        rng.choice(("none", "none", "none", "float", "f32", "mask")))
            c["idle"] = rng.choice((0, 0, 1, 2)) if c["B"] > 4 else 0
            # (the plain form holds all keys in fp32, padded to the longest sequence)
            fits = c["B"] * longest * Hkv * c["D"] <= 1 << 30 and c["B"] * longest * c["H"] <= 1 << 28 and c["H"] <= 128
        elif op == "write":
            c = _write(_log_int(rng, 1, 32768), rng.choice((1, 2, 3, 4, 8, 16)), rng.choice((32, 64, 128, 128, 256)), page, dtype,
                       rng.choice((0, 0, 2, 7)), rng.random() < 0.5, rng.choice((1, 4, 8)))
            fits = c["T"] * c["H"] * c["D"] <= 1 << 29
        elif op == "extend":
            c = _extend(_log_int(rng, 1, 2048), page, rng.choice((0, 1, 5)), _log_int(rng, 8, 8192),
                        rng.choice((1, 1, _log_int(rng, 2, 8192))))
            fits = c["B"] * c["new"] <= 1 << 20 and c["B"] * c["longest"] <= 1 << 24
        else:
            c = _release(_log_int(rng, 1, 2048), page, rng.choice((0, 1, 5)), _log_int(rng, 8, 32768), rng.choice((1, 2, 5, 40)))
            fits = c["B"] * c["longest"] <= 1 << 24
        if fits and work(c)["bytes"] <= most:
            return c


def _spread(n, lo, hi):
    """n whole numbers over lo .. hi, hi among them: the same for every seed (which shuffles them)."""
    return [hi - int((hi - lo + 1) * (i * 0.6180339887498949 % 1.0)) for i in range(n)]


def _lengths(case):
    n = case["B"] - case.get("idle", 0)
    return _spread(n, case["shortest"], case["longest"]) + [0] * case.get("idle", 0)


def _new_tokens(case):
    """New tokens of each request (in the order of _lengths, before the shuffle)."""
    return [1] * case["B"] if case["new"] == 1 else _spread(case["B"], 1, case["new"])


def _pages(tokens, page):
    return (tokens + page - 1) // page


def work(case):
    """What a pass cannot do without: the keys and values of all sequences (or the rows) once, what is asked of tables, the
    results once; 4 D operations for each pair of a query head and a key."""
    page = case["page"]
    if case["op"] == "attend":
        H, Hkv, D, lens = case["H"], case["Hkv"], case["D"], _lengths(case)
        keys = sum(lens)
        bias = {"none": 0, "float": 2 * H * keys, "f32": 4 * H * max(lens), "mask": keys}[case["bias"]]
        table = 4 * sum(_pages(n, page) for n in lens) + 4 * len(lens)
        return {"bytes": 4 * keys * Hkv * D + 4 * len(lens) * H * D + bias + table, "flops": 4 * H * D * keys}
    if case["op"] == "write":
        T = case["T"]
        rows = T - (len(range(0, T, case["skip"])) if case["skip"] else 0)
        return {"bytes": 8 * T + 8 * rows * case["Hkv"] * case["D"], "flops": 0}
    lens = _lengths(case)
    if case["op"] == "extend":
        new = _new_tokens(case)
        pages = sum(_pages(a + n, page) - _pages(a, page) for a, n in zip(lens, new))
        return {"bytes": 8 * sum(new) + 8 * pages + 12 * len(lens), "flops": 0}
    pages = sum(_pages(a, page) for a in lens[:: case["done"]])
    return {"bytes": 8 * pages + 9 * len(lens), "flops": 0}


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _table(rows, pages_of_each, order):
    """(B, rows) table whose rows begin with that many pages each, taken from `order` one after the other."""
    count = pages_of_each.long()
    at = torch.arange(rows, device="cuda")[None]
    place = count.cumsum(0)[:, None] - count[:, None] + at
    return torch.where(at < count[:, None], order[place.clamp(max=order.numel() - 1)], torch.zeros_like(place)).int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    page = case["page"]

    def normal(*shape, dtype, scale=1.0):
        t = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)
        return t.mul_(scale) if scale != 1.0 else t

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda")

    s = {"op": case["op"], "page": page}
    if case["op"] == "write":
        T, Hkv, H, D, dt = case["T"], case["Hkv"], case["H"], case["D"], _DTYPES[case["dtype"]]
        pages = _pages(T, page) + 3
        if case["packed"]:
            qkv = normal(T, H + 2 * Hkv, D, dtype=dt)
            s["k"], s["v"] = qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        else:
            s["k"], s["v"] = normal(T, Hkv, D, dtype=dt), normal(T, Hkv, D, dtype=dt)
        # (the plain form needs a page behind the cache for the rows that have no slot)
        s["k_room"], s["v_room"] = (normal(pages + 1, page, Hkv, D, dtype=dt) for _ in range(2))
        s["k_cache"], s["v_cache"] = s["k_room"][:pages], s["v_room"][:pages]
        at = torch.arange(T, device="cuda")
        s["slots"] = shuffled(pages)[at // page] * page + at % page
        if case["skip"]:
            s["slots"][:: case["skip"]] = -1
        return s

    order = shuffled(case["B"] - case.get("idle", 0))
    order = torch.cat([order, torch.arange(order.numel(), case["B"], device="cuda")])
    host_lens = _lengths(case)
    s["lens"] = _ints(host_lens)[order]
    held = (s["lens"] + page - 1) // page
    n_held = sum(_pages(n, page) for n in host_lens)
    if case["op"] == "attend":
        B, H, Hkv, D, dt = case["B"], case["H"], case["Hkv"], case["D"], _DTYPES[case["dtype"]]
        pages, width = n_held + 5, _pages(max(host_lens), page) + 1
        s["k_cache"], s["v_cache"] = normal(pages, page, Hkv, D, dtype=dt), normal(pages, page, Hkv, D, dtype=dt)
        s["q"] = normal(B, H, D, dtype=dt)
        s["table"] = _table(width, held, shuffled(pages))
        N = width * page
        s["bias"] = None
        if case["bias"] == "float":
            s["bias"] = normal(B, H, N, dtype=dt, scale=0.5)
        elif case["bias"] == "f32":
            s["bias"] = normal(H, N, dtype=torch.float32, scale=0.5)[None].expand(B, H, N)
        elif case["bias"] == "mask":
            keep = torch.empty((B, N), dtype=torch.uint8, device="cuda").random_(0, 10, generator=g).bool()
            s["bias"] = keep[:, None].expand(B, H, N)
        return s

    # tables: requests hold their pages, the others lie on the stack
    if case["op"] == "extend":
        host_new = _new_tokens(case)
        s["new"], s["num_tokens"] = _ints(host_new)[order], sum(host_new)
        more = sum(_pages(a + n, page) - _pages(a, page) for a, n in zip(host_lens, host_new))
        width = max(_pages(a + n, page) for a, n in zip(host_lens, host_new)) + 1
        pages = n_held + more + 7
        ids = shuffled(pages)
        s["table"] = _table(width, held, ids)
        s["free_pages"] = torch.cat([ids[n_held:], ids[:n_held]]).int()
        s["free_count"] = _ints([pages - n_held])
        return s
    width, pages = max(1, _pages(max(host_lens), page)), n_held + 7
    ids = shuffled(pages)
    s["table"] = _table(width, held, ids)
    s["free_pages"] = torch.cat([ids[n_held:], torch.zeros_like(ids[:n_held])]).int()
    s["free_count"] = _ints([pages - n_held])
    finished = torch.zeros(case["B"], dtype=torch.bool, device="cuda")
    finished[:: case["done"]] = True
    s["finished"] = finished[order]
    return s


# ------------------------------------------------------------------------------------- the operators
def run(s):
    if own:
        return _run_own(s)
    return {"attend": _plain_attend, "write": _plain_write, "extend": _plain_extend, "release": _plain_release}[s["op"]](s)


def _run_own(s):
    import triton_flashattn_b200 as fa

    if s["op"] == "attend":
        return fa.paged_attention_fn(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["bias"])
    if s["op"] == "write":
        fa.paged_kv_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if s["op"] == "extend":
        slots, lens, count = fa.paged_kv_extend(s["table"], s["lens"], s["new"], s["free_pages"], s["free_count"], s["page"],
                                                s["num_tokens"])
        return {"slots": slots, "lens": lens, "free_count": count, "table": s["table"]}
    lens, count = fa.paged_kv_release(s["table"], s["lens"], s["finished"], s["free_pages"], s["free_count"], s["page"])
    return {"lens": lens, "free_count": count, "free_pages": s["free_pages"]}


def _plain_attend(s):
    q, table, lens = s["q"], s["table"].long(), s["lens"].long()
    B, H, D = q.shape
    Hkv, N = s["k_cache"].shape[2], table.shape[1] * s["page"]
    k = s["k_cache"][table].reshape(B, N, Hkv, D).permute(0, 2, 3, 1).float()
    v = s["v_cache"][table].reshape(B, N, Hkv, D).permute(0, 2, 1, 3).float()
    score = (q.float().view(B, Hkv, H // Hkv, D) @ k).view(B, H, N) * D ** -0.5
    keep = (torch.arange(N, device=q.device) < lens[:, None])[:, None]
    if s["bias"] is not None:
        if s["bias"].dtype == torch.bool:
            keep = keep & s["bias"]
        else:
            score = score + s["bias"].float()
    score = torch.where(keep, score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, Hkv, H // Hkv, N) @ v).view(B, H, D)
    return (out / torch.where(total > 0, total, 1.0)).to(q.dtype)


def _plain_write(s):
    pages, page, Hkv, D = s["k_cache"].shape
    at = torch.where(s["slots"] >= 0, s["slots"], pages * page)
    for room, rows in ((s["k_room"], s["k"]), (s["v_room"], s["v"])):
        room.view(-1, Hkv * D).index_copy_(0, at, rows.reshape(-1, Hkv * D))
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_extend(s):
    page, T, table = s["page"], s["num_tokens"], s["table"]
    B, width = table.shape
    old, new, count = s["lens"].long(), s["new"].long().clamp(min=0), s["free_count"].long()
    end = new.cumsum(0)
    have = (old + page - 1) // page
    fits = (old + new <= width * page) & (end <= T)
    need = torch.where(fits, (old + new + page - 1) // page - have, 0)
    rank = need.cumsum(0) - need
    granted = fits & ((need == 0) | (rank + need <= count))
    # new pages, by their place in the row
    at = torch.arange(width, device=table.device)[None]
    j = at - have[:, None]
    fresh = granted[:, None] & (j >= 0) & (j < need[:, None])
    from_stack = s["free_pages"][(count - 1 - rank[:, None] - j).clamp(0, s["free_pages"].numel() - 1)]
    table.copy_(torch.where(fresh, from_stack, table))
    # slots, by token
    t = torch.arange(T, device=table.device)
    b = torch.searchsorted(end, t, right=True).clamp(max=B - 1)
    where = old[b] + t - (end - new)[b]
    slot = table[b, (where // page).clamp(max=width - 1)].long() * page + where % page
    slots = torch.where(granted[b] & (t < end[-1]), slot, -1)
    lens = torch.where(granted, old + new, old).int()
    return {"slots": slots, "lens": lens, "free_count": (count - torch.where(granted, need, 0).sum()).int(), "table": table}


def _plain_release(s):
    page, table, stack = s["page"], s["table"], s["free_pages"]
    lens, count = s["lens"].long(), s["free_count"].long()
    gone = torch.where(s["finished"], (lens + page - 1) // page, 0)
    end = gone.cumsum(0)
    # the stack by its places: which request's page comes to lie there
    i = torch.arange(stack.numel(), device=stack.device) - count
    b = torch.searchsorted(end, i, right=True).clamp(max=lens.numel() - 1)
    j = (i - (end - gone)[b]).clamp(0, table.shape[1] - 1)
    stack.copy_(torch.where((i >= 0) & (i < end[-1]), table[b, j], stack))
    left = torch.where(s["finished"], 0, lens).int()
    return {"lens": left, "free_count": (count + end[-1]).clamp(max=stack.numel()).int(), "free_pages": stack}


# ------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """Attention from its definition, sequence by sequence in 64 bits, and rows where they belong; the other operators move and
    count whole values."""
    if case["op"] not in ("attend", "write"):
        return None
    s = prepare(case, seed)
    if case["op"] == "write":
        has = s["slots"] >= 0
        out = {}
        for name in ("k", "v"):
            cache = s[name + "_cache"].double()
            cache[s["slots"][has] // case["page"], s["slots"][has] % case["page"]] = s[name][has].double()
            out[name + "_cache"] = cache
        return out
    H, Hkv, page = case["H"], case["Hkv"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        place = torch.arange(n, device="cuda")
        rows = s["table"][b].long()[place // page], place % page
        keys, values = s["k_cache"][rows].double(), s["v_cache"][rows].double()  # (n, Hkv, D)
        for h in range(Hkv):
            heads = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
            logits = s["q"][b, heads].double() @ keys[:, h].T / math.sqrt(case["D"])
            if case["bias"] == "mask":
                logits = logits.masked_fill(~s["bias"][b, heads, :n], -math.inf)
            elif case["bias"] != "none":
                logits = logits + s["bias"][b, heads, :n].double()
            weights = torch.softmax(logits, -1).nan_to_num(0.0)  # (a row that its mask leaves empty is 0)
            out[b, heads] = weights @ values[:, h]
    return out
