"""The paged-cache operators of this package, as cases that can be timed and compared.

Four operators of a step that serves many requests from a paged K/V cache:

  plan       block tables, slot maps and positions, built on the GPU from request lengths
  rotary     rotary positions with one or more axes over [batch, heads, seq_len, head_dim]
  append     rotary positions of a step's new Q and K, with K and V written to their cache slots
  attention  the new tokens' attention over the paged cache (one token a request, chunks, or both)

With `own` false every operator runs in its plain form: elementary torch operations in 32 bits (angles in 64),
rounded once at the end. With `own` true it runs as a user of the package calls it.
"""
import math

import numpy as np
import torch

own = False

AXES = {1: "64", 3: "16,24,24"}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _plan_case(name, seqs, decode, new_hi, cached_hi, page):
    return {"name": name, "op": "plan", "seqs": seqs, "decode": decode, "new_lo": 1, "new_hi": new_hi,
            "cached_lo": 0, "cached_hi": cached_hi, "page": page}


def _rotary_case(name, batch, heads, t, h, w, dim, sections, interleaved):
    return {"name": name, "op": "rotary", "batch": batch, "heads": heads, "t": t, "h": h, "w": w, "dim": dim,
            "sections": sections, "interleaved": interleaved}


def _append_case(name, seqs, decode, new_hi, cached_lo, cached_hi, heads, kv_heads, dim, page, sections):
    return {"name": name, "op": "append", "seqs": seqs, "decode": decode, "new_lo": 1, "new_hi": new_hi,
            "cached_lo": cached_lo, "cached_hi": cached_hi, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "sections": sections, "interleaved": False}


def _attention_case(name, seqs, decode, new_lo, new_hi, cached_lo, cached_hi, heads, kv_heads, dim, page):
    return {"name": name, "op": "attention", "seqs": seqs, "decode": decode, "new_lo": new_lo, "new_hi": new_hi,
            "cached_lo": cached_lo, "cached_hi": cached_hi, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page}


def listed():
    return [
        # One decode step of a small server: 16 requests, a token each. Latency counts.
        _plan_case("plan_decode_16", 16, 16, 1, 4096, 16),
        # A step that takes in prompts: 512 requests, up to 513 new tokens each, odd lengths.
        _plan_case("plan_prompts_512", 512, 128, 513, 8192, 16),
        # Image tokens (a 32 x 64 grid) of a small model, two images, height and width on axes of their own.
        _rotary_case("rotary_image_2048", 2, 8, 1, 32, 64, 64, "8,12,12", False),
        # Video tokens (16 x 32 x 32) with time, height and width, neighbouring elements as pairs.
        _rotary_case("rotary_video_16384", 1, 32, 16, 32, 32, 128, "16,24,24", True),
        # A decode step's new tokens: 64 requests far into their context.
        _append_case("append_decode_64", 64, 64, 1, 0, 131072, 32, 8, 128, 16, "64"),
        # Prompts with images: 16 requests, up to 1025 new tokens each, three position axes.
        _append_case("append_prompts_16", 16, 0, 1025, 0, 8192, 32, 8, 128, 64, "16,24,24"),
        # One user's decode step: the smallest call, where latency counts.
        _attention_case("attention_decode_1", 1, 1, 1, 1, 2047, 2047, 8, 8, 64, 16),
        # A decode step of 32 requests with ragged contexts and grouped heads.
        _attention_case("attention_decode_32", 32, 32, 1, 1, 17, 4096, 32, 8, 128, 16),
        # A large decode step: 64 requests with long ragged contexts.
        _attention_case("attention_decode_64_long", 64, 64, 1, 1, 4095, 16384, 32, 8, 128, 64),
        # Verification of drafted tokens: 16 requests of 5 to 8 new tokens each.
        _attention_case("attention_draft_16", 16, 0, 5, 8, 1000, 8192, 32, 8, 128, 16),
        # A chunk of a long prompt: 2048 new tokens behind 14336 cached ones.
        _attention_case("attention_chunk_2048", 1, 0, 2048, 2048, 14336, 14336, 32, 8, 128, 64),
        # A mixed step: 20 requests decode while 4 bring in prompt chunks of odd sizes.
        _attention_case("attention_mixed_24", 24, 20, 100, 700, 1, 2500, 16, 16, 64, 32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _plain_cost(case):
    """Elements of the plain attention's scores and of its gathered keys."""
    cached, new = _lengths(case)
    longest = _pages(int((cached + new).max()), case["page"]) * case["page"]
    return (case["seqs"] * case["heads"] * int(new.max()) * longest,
            case["seqs"] * case["kv_heads"] * longest * case["dim"])


def draw(rng):
    op = rng.choice(["plan", "rotary", "append", "attention", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        seqs = _log(rng, 1, 512)
        return _plan_case("", seqs, rng.randint(0, seqs), _log(rng, 1, 513), _log(rng, 16, 8192), page)
    dim = rng.choice([64, 128])
    if op == "rotary":
        pairs = dim // 2
        a = rng.randint(1, pairs // 2)
        b = rng.randint(1, pairs - a - 1)
        h, w = rng.randint(1, 40), rng.randint(1, 40)
        t = _log(rng, 1, max(1, 16384 // (h * w)))
        return _rotary_case("", rng.randint(1, 2), rng.randint(1, 16), t, h, w, dim,
                            "%d,%d,%d" % (a, b, pairs - a - b), rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    if op == "append":
        seqs = _log(rng, 1, 64)
        sections = "%d" % (dim // 2) if rng.random() < 0.5 else "%d,%d,%d" % (dim // 8, dim // 8, dim // 4)
        return _append_case("", seqs, rng.randint(0, seqs), _log(rng, 1, 8192 // seqs), 0, _log(rng, 1, 131072),
                            heads, kv_heads, dim, page, sections)
    while True:
        seqs = _log(rng, 1, 64)
        kind = rng.choice(["decode", "draft", "chunk", "mixed"])
        decode = seqs if kind == "decode" else rng.randint(0, seqs - 1) if kind == "mixed" else 0
        new_hi = 1 if kind == "decode" else rng.randint(2, 12) if kind == "draft" else _log(rng, 2, 2048)
        case = _attention_case("", seqs, decode, 1, new_hi, 0, _log(rng, 16, 16384), heads, kv_heads, dim, page)
        scores, keys = _plain_cost(case)
        if scores <= 1.2e9 and keys <= 1.1e9 and work(case)["flops"] <= 5e11:
            return case


# ---------------------------------------------------------------------------
# Lengths and sizes: the same for every seed up to their order
# ---------------------------------------------------------------------------
def _lengths(case):
    """(cached, new) of each request: spread evenly over their ranges, the first `decode` with one new token."""
    i = np.arange(1, case["seqs"] + 1)
    u = (i * 0.6180339887498949) % 1.0
    v = (i * 0.7548776662466927) % 1.0
    cached = case["cached_lo"] + np.floor((case["cached_hi"] - case["cached_lo"] + 1) * u).astype(np.int64)
    new = case["new_lo"] + np.floor((case["new_hi"] - case["new_lo"] + 1) * v).astype(np.int64)
    new[: case["decode"]] = 1
    return cached, new


def _pages(tokens, page):
    return -(-tokens // page)


def _sections(case):
    return tuple(int(x) for x in case["sections"].split(","))


def work(case):
    if case["op"] == "rotary":
        tokens = case["t"] * case["h"] * case["w"]
        n = case["batch"] * case["heads"] * tokens * case["dim"]
        return {"bytes": 4 * n + 4 * tokens * len(_sections(case)) + 2 * case["dim"], "flops": 3 * n}
    cached, new = _lengths(case)
    total, kv = int(new.sum()), cached + new
    if case["op"] == "plan":
        taken = int((_pages(kv, case["page"]) - _pages(cached, case["page"])).sum())
        # lengths in; starts, total lengths, positions and slots out; a page id read and written per new page
        return {"bytes": 16 * case["seqs"] + 8 * total + 8 * taken, "flops": 0}
    rows = case["heads"] + 2 * case["kv_heads"]
    if case["op"] == "append":
        return {"bytes": 4 * total * rows * case["dim"] + 4 * total * (len(_sections(case)) + 1),
                "flops": 3 * total * (case["heads"] + case["kv_heads"]) * case["dim"]}
    pairs = int((new * cached + new * (new + 1) // 2).sum())
    return {"bytes": 4 * total * case["heads"] * case["dim"] + 4 * int(kv.sum()) * case["kv_heads"] * case["dim"]
                     + 4 * int(_pages(kv, case["page"]).sum()),
            "flops": 4 * case["heads"] * case["dim"] * pairs}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _requests(case, seed, gen):
    """Request lengths in a shuffled order, a table that holds the cached pages, and the list of free pages."""
    order = np.random.RandomState(seed).permutation(case["seqs"])
    cached, new = (x[order] for x in _lengths(case))
    page = case["page"]
    have, want = _pages(cached, page), _pages(cached + new, page)
    num_pages = int(want.sum()) + 8
    width = int(want.max()) + 1
    ids = torch.randperm(num_pages, generator=gen, device="cuda").to(torch.int32)
    have_t = torch.from_numpy(have).cuda()
    column = torch.arange(width, device="cuda")
    held = column < have_t[:, None]
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda")
    table[held] = ids[: int(have.sum())]
    return {
        "cached": torch.from_numpy(cached).to("cuda", torch.int32), "new": torch.from_numpy(new).to("cuda", torch.int32),
        "table": table, "free_pages": ids[int(have.sum()):].clone(),
        "cursor": torch.zeros(1, dtype=torch.int32, device="cuda"),
        "total": int(new.sum()), "max_new": int(new.max()), "num_pages": num_pages, "page": page,
    }


def _small_cache(case, seed, gen):
    """As _requests, for a cache that holds the new tokens' pages alone: earlier pages are other steps' work."""
    state = _requests({**case, "cached_hi": min(case["cached_hi"], 64), "cached_lo": 0}, seed, gen)
    order = np.random.RandomState(seed).permutation(case["seqs"])
    cached, new = (torch.from_numpy(x[order]).cuda() for x in _lengths(case))
    start = torch.cumsum(new, 0) - new
    at = torch.arange(state["total"], device="cuda")
    far = torch.repeat_interleave(cached - start, new, output_size=state["total"]) + at
    axes = len(_sections(case))
    if axes == 1:
        state["positions"] = far[None].to(torch.int32)
    else:   # one axis counts tokens, the others rows and columns of 32-wide images
        state["positions"] = torch.stack([far, (at // 32) % 32, at % 32][:axes]).to(torch.int32)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)

    def frequencies(dim):
        return 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float32) / dim)

    op = case["op"]
    if op == "rotary":
        t, h, w = case["t"], case["h"], case["w"]
        at = torch.arange(t * h * w, device="cuda") + seed % 7
        return {"op": op, "x": normal(case["batch"], case["heads"], t * h * w, case["dim"]),
                "positions": torch.stack([at // (h * w), (at // w) % h, at % w]).to(torch.int32),
                "inv_freq": frequencies(case["dim"]), "sections": _sections(case), "interleaved": case["interleaved"]}
    if op == "plan":
        state = _requests(case, seed, gen)
        state.update(op=op, heads=8, kv_heads=8, dim=64)
        return state
    state = _small_cache(case, seed, gen) if op == "append" else _requests(case, seed, gen)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    state.update(op=op, heads=heads, kv_heads=kv_heads, dim=dim)
    state["k_cache"] = normal(state["num_pages"], kv_heads, case["page"], dim)
    state["v_cache"] = normal(state["num_pages"], kv_heads, case["page"], dim)
    # The step's plan: a program builds it once and every layer's calls use it.
    if own:
        state["plan"] = _plan_own(state)
        state["slots"] = state["plan"].slots
    else:
        state["plan"] = _plan_plain(state)
        state["table"].copy_(state["plan"]["block_table"])
        state["slots"] = state["plan"]["slots"]
    if op == "append":
        # A fused projection's output: Q, K and V of a token side by side.
        qkv = normal(state["total"], heads + 2 * kv_heads, dim)
        state["q"], state["k"], state["v"] = qkv.split([heads, kv_heads, kv_heads], dim=1)
        state.update(inv_freq=frequencies(dim), sections=_sections(case), interleaved=case["interleaved"])
    else:
        state["q"] = normal(state["total"], heads, dim)
    return state


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _plan_plain(s):
    cached, new, page, table = s["cached"].long(), s["new"].long(), s["page"], s["table"]
    kv = cached + new
    ends = torch.cumsum(new, 0)
    start = torch.cat([torch.zeros_like(ends[:1]), ends])
    seq = torch.repeat_interleave(torch.arange(new.numel(), device=new.device), new, output_size=s["total"])
    positions = cached[seq] + torch.arange(s["total"], device=new.device) - start[seq]
    have, want = (cached + page - 1) // page, (kv + page - 1) // page
    first = torch.cumsum(want - have, 0) - (want - have) + s["cursor"].long()
    column = torch.arange(table.shape[1], device=new.device)
    taken = (column >= have[:, None]) & (column < want[:, None])
    source = (first[:, None] + column - have[:, None]).clamp(0, s["free_pages"].numel() - 1)
    table = torch.where(taken, s["free_pages"][source], table)
    slots = table[seq, positions // page].long() * page + positions % page
    return {"query_start": start.int(), "kv_lens": kv.int(), "positions": positions.int(), "slots": slots.int(),
            "block_table": table, "free_cursor": (s["cursor"] + (want - have).sum()).int()}


def _angles(positions, inv_freq, sections):
    """cos and sin of each token's angles, [..., tokens, pairs] from positions [axes, ..., tokens]: angles in 64 bits."""
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(positions.device)
    angle = positions[axis].double().movedim(0, -1) * inv_freq.double()
    return torch.cos(angle).float(), torch.sin(angle).float()


def _rotate(x, cos, sin, interleaved):
    """x [..., pairs * 2] rotated; cos and sin broadcast over x's leading dimensions."""
    x = x.float()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, dim=-1)
    c, d = a * cos - b * sin, b * cos + a * sin
    return torch.stack([c, d], dim=-1).flatten(-2) if interleaved else torch.cat([c, d], dim=-1)


def _rotary_plain(s):
    cos, sin = _angles(s["positions"], s["inv_freq"], s["sections"])
    return _rotate(s["x"], cos, sin, s["interleaved"]).to(torch.bfloat16)


def _append_plain(s):
    cos, sin = _angles(s["positions"], s["inv_freq"], s["sections"])
    cos, sin = cos[:, None], sin[:, None]
    q = _rotate(s["q"], cos, sin, s["interleaved"]).to(torch.bfloat16)
    k = _rotate(s["k"], cos, sin, s["interleaved"]).to(torch.bfloat16)
    page, row = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    s["k_cache"][page, :, row] = k
    s["v_cache"][page, :, row] = s["v"]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention_plain(s):
    table, heads, kv_heads, dim = s["table"].long().clamp(min=0), s["heads"], s["kv_heads"], s["dim"]
    seqs, most, group = table.shape[0], s["max_new"], heads // kv_heads
    length = table.shape[1] * s["page"]
    new, cached = s["new"].long(), s["cached"].long()

    def gathered(cache):
        return cache[table].permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, length, dim).float()

    step = torch.arange(most, device=table.device)
    real = step < new[:, None]
    rows = (torch.cumsum(new, 0) - new)[:, None] + step
    q = s["q"][rows.clamp(max=s["total"] - 1)].float()
    q = q.reshape(seqs, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, group * most, dim)
    scores = torch.matmul(q, gathered(s["k_cache"]).transpose(-1, -2)).mul_(1.0 / math.sqrt(dim))
    scores = scores.view(seqs, kv_heads, group, most, length)
    hidden = torch.arange(length, device=table.device) > (cached[:, None] + step)[:, :, None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1)
    out = torch.matmul(scores.view(seqs, kv_heads, group * most, length), gathered(s["v_cache"]))
    out = out.view(seqs, kv_heads, group, most, dim) / total[..., None]
    return out.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, dim)[real].to(torch.bfloat16)


# ---------------------------------------------------------------------------
# The package's calls
# ---------------------------------------------------------------------------
def _plan_own(s):
    import cuda_fused_attention_b200 as fa
    return fa.paged_plan(s["cached"], s["new"], s["table"], s["free_pages"], s["total"],
                         fa.PagedShape(s["heads"], s["kv_heads"], s["dim"], s["page"]), s["num_pages"],
                         free_cursor=s["cursor"], max_new=s["max_new"])


def _run_own(s):
    import cuda_fused_attention_b200 as fa
    if s["op"] == "plan":
        p = _plan_own(s)
        return {"query_start": p.query_start, "kv_lens": p.kv_lens, "positions": p.positions, "slots": p.slots,
                "block_table": s["table"], "free_cursor": p.free_cursor}
    if s["op"] == "rotary":
        return fa.rotary_embed(s["x"], s["positions"], s["inv_freq"], sections=s["sections"],
                               interleaved=s["interleaved"])
    if s["op"] == "append":
        q = fa.rotary_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["positions"], s["slots"],
                             s["inv_freq"], sections=s["sections"], interleaved=s["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return fa.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["plan"])


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "plan":
        return _plan_plain(state)
    if state["op"] == "rotary":
        return _rotary_plain(state)
    if state["op"] == "append":
        return _append_plain(state)
    return _attention_plain(state)


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _turned(x, positions, inv_freq, sections, interleaved):
    """x [tokens, heads, dim] with each pair, read as a complex number, turned by its angle."""
    x, pairs = x.double(), x.shape[-1] // 2
    at = torch.empty(x.shape[0], pairs, dtype=torch.float64, device=x.device)
    lo = 0
    for a, n in enumerate(sections):
        at[:, lo:lo + n] = positions[a].double()[:, None] * inv_freq.double()[lo:lo + n]
        lo += n
    turn = torch.polar(torch.ones_like(at), at)[:, None]
    index = torch.arange(pairs, device=x.device)
    re, im = (2 * index, 2 * index + 1) if interleaved else (index, index + pairs)
    z = torch.complex(x[..., re].contiguous(), x[..., im].contiguous()) * turn
    out = torch.empty_like(x)
    out[..., re], out[..., im] = z.real, z.imag
    return out


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "rotary":
        batch, heads, tokens, dim = s["x"].shape
        flat = s["x"].permute(2, 0, 1, 3).reshape(tokens, batch * heads, dim)
        out = _turned(flat, s["positions"], s["inv_freq"], s["sections"], s["interleaved"])
        return out.view(tokens, batch, heads, dim).permute(1, 2, 0, 3).contiguous()
    if case["op"] == "append":
        how = (s["positions"], s["inv_freq"], s["sections"], s["interleaved"])
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        slots, page = s["slots"].cpu().numpy().astype(np.int64), case["page"]
        at = torch.from_numpy(slots // page).cuda(), torch.from_numpy(slots % page).cuda()
        k_cache[at[0], :, at[1]] = _turned(s["k"], *how)
        v_cache[at[0], :, at[1]] = s["v"].double()
        return {"q": _turned(s["q"], *how), "k_cache": k_cache, "v_cache": v_cache}
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group, out, row = heads // kv_heads, [], 0
    table = s["table"].cpu().numpy()
    for b, (cached, new) in enumerate(zip(s["cached"].tolist(), s["new"].tolist())):
        pages = torch.from_numpy(table[b, : _pages(cached + new, page)].astype(np.int64)).cuda()
        last = torch.arange(cached, cached + new, device="cuda")[:, None]
        seen = torch.arange(cached + new, device="cuda")[None] <= last
        o = torch.empty(new, heads, dim, dtype=torch.float64, device="cuda")
        for h in range(kv_heads):
            k = s["k_cache"][pages, h].reshape(-1, dim)[: cached + new].double()
            v = s["v_cache"][pages, h].reshape(-1, dim)[: cached + new].double()
            for g in range(h * group, (h + 1) * group):
                x = s["q"][row: row + new, g].double() @ k.T / math.sqrt(dim)
                o[:, g] = torch.softmax(torch.where(seen, x, -math.inf), -1) @ v
        out.append(o)
        row += new
    return torch.cat(out)
