"""Steps over a paged K/V cache held in 8 bits, as cases that can be timed and checked.

  append   a step's new K and V rows rotated to their positions, quantised and
           put into their page slots, q rotated with them, and the rows read
           back as the values the cache now holds (KVPool.rope_kv_append and
           kv_read, or their prefill forms)
  decode   attention of one new token per sequence over the cache (KVPool.decode)
  prefill  causal attention of chunks of prompts over the cache, packed rows
           (KVPool.prefill)

The cache is one uint8 tensor [pages][layers][kv_heads][record], a record holding
16 tokens of one K/V head: K codes int8 [4][hdp/16][4][16] (four tokens of sixteen
dimensions lie together), V codes int8 [hdp][16], then 16 K scales and 16 V scales
in fp32; hdp is the head size rounded up to a multiple of 16.  A value is its code
times the scale of its token and head: scale = max|x| / 127 in fp32, code =
rint(x * fp32(127 / max|x|)), the product taken exactly.

Lengths are drawn from the case's own "lengths" number, so they are part of the
case; values and page ids come from the seed.  K, V and q are N(0, 1), as behind a
norm.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16

H12X64 = {"heads": 12, "kv_heads": 12, "head_dim": 64}
H32X128 = {"heads": 32, "kv_heads": 32, "head_dim": 128}
H32_8X128 = {"heads": 32, "kv_heads": 8, "head_dim": 128}
H16X96 = {"heads": 16, "kv_heads": 16, "head_dim": 96}


def listed():
    return [
        # one user generating through a small model's layer: latency is everything
        {"name": "append_1", "kind": "append", "form": "decode", **H12X64, "layers": 2, "batch": 1,
         "cached_min": 255, "cached_max": 255, "new_min": 1, "new_max": 1, "lengths": 0},
        # a decode step's rows of a 7B-shaped model's layer
        {"name": "append_64", "kind": "append", "form": "decode", **H32X128, "layers": 1, "batch": 64,
         "cached_min": 0, "cached_max": 1000, "new_min": 1, "new_max": 1, "lengths": 1},
        # chunks of prompts that begin and end inside pages, head size no power of two
        {"name": "append_chunks_head96", "kind": "append", "form": "prefill", **H16X96, "layers": 2, "batch": 6,
         "cached_min": 0, "cached_max": 333, "new_min": 50, "new_max": 700, "lengths": 2},
        # long fresh prompts through a 7B-shaped model's layer: bytes are everything
        {"name": "append_4_prompts_4096", "kind": "append", "form": "prefill", **H32X128, "layers": 1, "batch": 4,
         "cached_min": 0, "cached_max": 0, "new_min": 4096, "new_max": 4096, "lengths": 3},
        # one user's token over a short context
        {"name": "decode_1_ctx256", "kind": "decode", **H12X64, "layers": 2, "batch": 1,
         "ctx_min": 256, "ctx_max": 256, "lengths": 4},
        # a serving batch of unequal contexts
        {"name": "decode_32_mixed", "kind": "decode", **H12X64, "layers": 2, "batch": 32,
         "ctx_min": 16, "ctx_max": 1024, "lengths": 5},
        # grouped-query heads over retrieved documents of many lengths
        {"name": "decode_24_gqa", "kind": "decode", **H32_8X128, "layers": 1, "batch": 24,
         "ctx_min": 512, "ctx_max": 8192, "lengths": 6},
        # the largest decode: 64 long contexts, a K/V head per query head
        {"name": "decode_64_ctx4096", "kind": "decode", **H32X128, "layers": 1, "batch": 64,
         "ctx_min": 4096, "ctx_max": 4096, "lengths": 7},
        # one very long document, split over the GPU
        {"name": "decode_1_ctx131072", "kind": "decode", **H32_8X128, "layers": 1, "batch": 1,
         "ctx_min": 131072, "ctx_max": 131072, "lengths": 8},
        # eight fresh prompts through a small model's layer
        {"name": "prefill_8_prompts", "kind": "prefill", **H12X64, "layers": 2, "batch": 8,
         "cached_min": 0, "cached_max": 0, "new_min": 128, "new_max": 1024, "lengths": 9},
        # chunked prefill behind cached tokens, grouped-query heads
        {"name": "prefill_4_chunks_gqa", "kind": "prefill", **H32_8X128, "layers": 1, "batch": 4,
         "cached_min": 0, "cached_max": 4096, "new_min": 384, "new_max": 512, "lengths": 10},
        # one long prompt of a 7B-shaped model: products are everything
        {"name": "prefill_1_8192", "kind": "prefill", **H32X128, "layers": 1, "batch": 1,
         "cached_min": 0, "cached_max": 0, "new_min": 8192, "new_max": 8192, "lengths": 11},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_once(rng):
    heads, kv_heads, head_dim = rng.choice(
        [(12, 12, 64), (12, 12, 64), (32, 32, 128), (32, 8, 128), (32, 8, 128), (32, 4, 64), (14, 2, 64), (16, 16, 96),
         (32, 32, 80), (16, 8, 256), (6, 3, 36), (32, 1, 128)])
    case = {"kind": rng.choice(["append", "decode", "decode", "prefill"]), "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "layers": rng.randint(1, 3), "lengths": rng.randrange(1 << 30)}
    if case["kind"] == "decode":
        top = _log_int(rng, 1, 65536)
        return {**case, "batch": _log_int(rng, 1, 64), "ctx_min": _log_int(rng, max(1, top // 16), top), "ctx_max": top}
    cached = rng.choice([0, _log_int(rng, 1, 4096)])
    spans = {"cached_min": cached // 4, "cached_max": cached}
    if case["kind"] == "append" and rng.random() < 0.5:
        return {**case, "form": "decode", "batch": _log_int(rng, 1, 256), **spans, "new_min": 1, "new_max": 1}
    top = _log_int(rng, 1, 4096)
    new = {"new_min": _log_int(rng, max(1, top // 8), top), "new_max": top}
    if case["kind"] == "append":
        case["form"] = "prefill"
    return {**case, "batch": _log_int(rng, 1, 16), **spans, **new}


def draw(rng):
    most = {"append": 5e8, "decode": 2.3e9, "prefill": 1e9}
    while True:
        case = _draw_once(rng)
        w = work(case)
        padded = case["batch"] * case["heads"] * case.get("new_max", 1) * (
            case["ctx_max"] if case["kind"] == "decode" else case["cached_max"] + case["new_max"])
        if w["bytes"] <= most[case["kind"]] and w["flops"] <= 5.5e11 and (case["kind"] == "append" or padded <= 2.2e9):
            return case


# ------------------------------------------------------------------ lengths

def _ints(case, low, high, salt=0):
    r = random.Random(case["lengths"] * 3 + salt)
    return [r.randint(low, high) for _ in range(case["batch"])]


def _spans(case):
    """(first position, rows) of each sequence's new rows."""
    if case["kind"] == "decode":
        return [(n - 1, 1) for n in _ints(case, case["ctx_min"], case["ctx_max"])]
    return list(zip(_ints(case, case["cached_min"], case["cached_max"], 1), _ints(case, case["new_min"], case["new_max"])))


def _padded(head_dim):
    return (head_dim + 15) // 16 * 16


def work(case):
    spans = _spans(case)
    rows = sum(n for _, n in spans)
    H, G, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":  # q in and out, k and v in, codes and scales out, the values read back
        return {"bytes": rows * (8 * H * hd + 8 * G * hd + 2 * G * hd + 8 * G + 8 * G * hd), "flops": rows * (6 * (H + G) * hd + 6 * G * hd)}
    keys = sum(s + n for s, n in spans)
    pairs = sum(n * s + n * (n + 1) // 2 for s, n in spans)
    return {"bytes": keys * G * (2 * hd + 8) + 8 * rows * H * hd, "flops": 4 * pairs * H * hd}


# ------------------------------------------------------------------- inputs

def prepare(case, seed):
    spans = _spans(case)
    G, hd, L, B = case["kv_heads"], case["head_dim"], case["layers"], case["batch"]
    hdp, dev = _padded(hd), "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    pages = [(s + n + PAGE - 1) // PAGE for s, n in spans]
    max_pages, total = max(pages), sum(pages) + 3
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    tables = torch.zeros((B, max_pages), dtype=torch.int32)
    used = 0
    for b, n in enumerate(pages):
        tables[b, :n] = ids[used:used + n]
        used += n
    record = 32 * hdp + 8 * PAGE
    cache = torch.zeros((total, L, G, record), dtype=torch.uint8, device=dev)
    if case["kind"] != "append":  # what earlier steps left: codes of N(0, 1) rows, in every slot
        step = max(1, (1 << 28) // (L * G * record))
        for p in range(0, total, step):
            part = cache[p:p + step]
            codes = part[..., :32 * hdp].view(torch.int8)
            codes.copy_(torch.randn(codes.shape, generator=g, device=dev).mul_(45).round_().clamp_(-127, 127))
            if hdp > hd:  # the padding is zero
                k = _k_codes(part, hdp)
                for d in range(hd, hdp):
                    k[..., d // 16, :, d % 16] = 0
                _v_codes(part, hdp)[..., hd:, :] = 0
            scales = part[..., 32 * hdp:].view(torch.float32)
            scales.copy_(torch.rand(scales.shape, generator=g, device=dev).mul_(0.008).add_(0.018))
    rows = sum(n for _, n in spans)
    state = {"case": case, "cache": cache, "layer": L - 1, "tables": tables.to(dev)}
    state["q"] = torch.randn((rows, case["heads"] * hd), generator=g, device=dev)
    state["seq"] = torch.repeat_interleave(torch.arange(B), torch.tensor([n for _, n in spans])).to(dev)
    state["pos"] = torch.cat([torch.arange(s, s + n) for s, n in spans]).to(dev)
    state["spans"] = spans
    if case["kind"] == "append":
        state["k"], state["v"] = (torch.randn((rows, G * hd), generator=g, device=dev) for _ in range(2))
        top = max(s + n for s, n in spans)
        angle = torch.arange(top, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)
        state["cos"], state["sin"] = angle.cos().float().to(dev), angle.sin().float().to(dev)
        state["k_out"], state["v_out"] = torch.empty_like(state["k"]), torch.empty_like(state["v"])
    else:
        state["out"] = torch.empty_like(state["q"])
    # where the packed rows of a padded batch lie, and which of its places are rows
    most = max(n for _, n in spans)
    state["real"] = (torch.arange(most)[None] < torch.tensor([n for _, n in spans])[:, None]).to(dev)
    if own:  # the pool over the cache, and the step's batch uploaded, as a program keeps them over its layers
        import nitrorag_amd as na

        pool = na.KVPool.wrap_q8(cache, hd)
        if case["kind"] == "prefill" or case.get("form") == "prefill":
            pool.upload_prefill_batch(tables.numpy(), [s for s, _ in spans], [n for _, n in spans])
        else:
            pool.upload_decode_batch(tables.numpy(), [s for s, _ in spans])
        state["pool"] = pool
    return state


def _k_codes(cache, hdp):
    return cache[..., :16 * hdp].view(torch.int8).unflatten(-1, (4, hdp // 16, 4, 16))


def _v_codes(cache, hdp):
    return cache[..., 16 * hdp:32 * hdp].view(torch.int8).unflatten(-1, (hdp, 16))


def _scales(cache, hdp):
    return cache[..., 32 * hdp:].view(torch.float32).unflatten(-1, (2, 16))


# --------------------------------------------------------------------- runs

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state)
    return _append(state) if kind == "append" else _attend(state)


def _own(state):
    case, pool, layer = state["case"], state["pool"], state["layer"]
    shape = (case["heads"], case["kv_heads"], case["head_dim"])
    if case["kind"] == "append":
        q, k = state["q"].clone(), state["k"].clone()  # rotated in place
        prefill = case["form"] == "prefill"
        (pool.rope_kv_append_prefill if prefill else pool.rope_kv_append)(layer, q, k, state["v"], state["cos"], state["sin"], *shape)
        (pool.kv_read_prefill if prefill else pool.kv_read)(layer, state["k_out"], state["v_out"])
        return {"q": q, "k": state["k_out"], "v": state["v_out"]}
    (pool.prefill if case["kind"] == "prefill" else pool.decode)(layer, state["q"], state["out"], *shape)
    return {"out": state["out"]}


def _rotate(x, cos, sin):
    """Pairs (2i, 2i + 1) of rows [rows][heads][head_dim], in 64 bits, rounded once."""
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    c, s = cos[:, None].double(), sin[:, None].double()
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2).float()


def _quantise(x):
    """int8 codes and the fp32 scale of each row [rows][heads][head_dim]."""
    top = x.abs().amax(-1).double()
    scale = (top / torch.full_like(top, 127)).float()
    inverse = (torch.full_like(top, 127) / top).float()
    return torch.round(x.double() * inverse.double()[..., None]).to(torch.int8), scale


def _append(state):
    case, cache = state["case"], state["cache"][:, state["layer"]]
    hd, hdp, pos = case["head_dim"], _padded(case["head_dim"]), state["pos"]
    cos, sin = state["cos"][pos], state["sin"][pos]
    q = _rotate(state["q"].unflatten(-1, (-1, hd)), cos, sin).flatten(1)
    k, k_scale = _quantise(_rotate(state["k"].unflatten(-1, (-1, hd)), cos, sin))
    v, v_scale = _quantise(state["v"].unflatten(-1, (-1, hd)))
    k, v = (torch.nn.functional.pad(t, (0, hdp - hd)) for t in (k, v))
    page, slot = state["tables"][state["seq"], pos // PAGE].long(), pos % PAGE
    k_codes, v_codes, scales = _k_codes(cache, hdp), _v_codes(cache, hdp), _scales(cache, hdp)
    k_codes.permute(0, 2, 4, 1, 3, 5)[page, slot // 4, slot % 4] = k.unflatten(-1, (-1, 16))
    v_codes.permute(0, 3, 1, 2)[page, slot] = v
    scales.permute(0, 3, 1, 2)[page, slot] = torch.stack((k_scale, v_scale), -1)
    codes = k_codes.permute(0, 2, 4, 1, 3, 5)[page, slot // 4, slot % 4].flatten(-2), v_codes.permute(0, 3, 1, 2)[page, slot]
    held = scales.permute(0, 3, 1, 2)[page, slot]
    return {"q": q, "k": (codes[0][..., :hd].float() * held[..., :1]).flatten(1),
            "v": (codes[1][..., :hd].float() * held[..., 1:]).flatten(1)}


def _gathered(state):
    """K and V of every sequence in fp32, [batch][kv_heads][tokens][head_dim]."""
    hd, hdp = state["case"]["head_dim"], _padded(state["case"]["head_dim"])
    got = state["cache"][:, state["layer"]][state["tables"].long()]  # [batch][pages][kv_heads][record]
    k = _k_codes(got, hdp).permute(0, 2, 1, 3, 5, 4, 6).flatten(5).flatten(2, 4)
    v = _v_codes(got, hdp).permute(0, 2, 1, 4, 3).flatten(2, 3)
    s = _scales(got, hdp).permute(0, 2, 3, 1, 4).flatten(3)  # [batch][kv_heads][2][tokens]
    return k[..., :hd].float() * s[:, :, 0, :, None], v[..., :hd].float() * s[:, :, 1, :, None]


def _attend(state):
    case = state["case"]
    H, G, hd, real = case["heads"], case["kv_heads"], case["head_dim"], state["real"]
    k, v = _gathered(state)
    B, N = real.shape
    q = torch.zeros((B, N, H * hd), device=k.device)
    q[real] = state["q"]
    at = torch.full((B, N), 0, device=k.device)
    at[real] = state["pos"]
    # the query heads of a K/V head are rows of its product
    q = q.view(B, N, G, H // G, hd).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * N, hd)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(hd))
    hidden = torch.arange(k.shape[2], device=k.device)[None, None] > at[:, :, None]
    s = s.view(B, G, H // G, N, -1).masked_fill_(hidden[:, None, None], -math.inf).view(B, G, H // G * N, -1)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    out = out.view(B, G, H // G, N, hd).permute(0, 3, 1, 2, 4).reshape(B, N, H * hd)
    return {"out": out[real]}


# -------------------------------------------------------------------- exact

def exact(case, seed):
    """The same in 64 bits, a sequence and a head at a time.  The scale that a row
    is held with, its inverse and the rotated rows are fp32 numbers by definition."""
    state = prepare(case, seed)
    G, R, hd = case["kv_heads"], case["heads"] // case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":
        cos, sin = (state[n].double()[state["pos"]].repeat_interleave(2, -1)[:, None] for n in ("cos", "sin"))

        def turned(x):
            x = x.view(x.shape[0], -1, hd).double()
            other = torch.empty_like(x)
            other[..., 0::2], other[..., 1::2] = -x[..., 1::2], x[..., 0::2]
            return (x * cos + other * sin).to(torch.float32).double()

        def held(x):
            top = torch.maximum(x.max(-1).values, -x.min(-1).values)[..., None]
            inverse = torch.div(torch.tensor(127.0, dtype=torch.float64, device=x.device).expand_as(top), top).float().double()
            scale = torch.div(top, torch.tensor(127.0, dtype=torch.float64, device=x.device).expand_as(top)).float().double()
            return (torch.round(x * inverse) * scale).reshape(x.shape[0], -1)

        v = state["v"].view(-1, G, hd).double()
        return {"q": turned(state["q"]).reshape(len(v), -1), "k": held(turned(state["k"])), "v": held(v)}
    hdp, row, out = _padded(hd), 0, []
    layer = state["cache"][:, state["layer"]]
    for b, (start, n) in enumerate(state["spans"]):
        keys = start + n
        t = torch.arange(keys, device="cuda")
        page, slot = state["tables"][b].long()[t // PAGE], t % PAGE
        d = torch.arange(hd, device="cuda")
        q = state["q"][row:row + n].double().view(n, G, R, hd)
        row += n
        heads = []
        for g in range(G):
            rec = layer[page, g]  # [keys][record]
            scale = rec[:, 32 * hdp:].contiguous().view(torch.float32).double()
            k_at = (slot[:, None] // 4) * 4 * hdp + (d[None] // 16) * 64 + (slot[:, None] % 4) * 16 + d[None] % 16
            v_at = 16 * hdp + d[None] * 16 + slot[:, None]
            codes = rec.view(torch.int8)
            k = codes.gather(1, k_at).double() * scale.gather(1, slot[:, None])
            v = codes.gather(1, v_at).double() * scale.gather(1, 16 + slot[:, None])
            for r in range(R):
                s = q[:, g, r] @ k.t().contiguous() / math.sqrt(hd)
                s = s.masked_fill(t[None] > (start + torch.arange(n, device="cuda"))[:, None], -math.inf)
                heads.append(torch.softmax(s, -1) @ v)
        out.append(torch.stack(heads, 1).reshape(n, -1))
    return {"out": torch.cat(out)}
