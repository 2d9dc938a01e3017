"""Timed cases of the rotation, paged-append and shared-prefix attention operators.

`run` computes a case in its plain form (elementary torch operations, 32 bits and more)
or, with `own` set, through the framework's public calls.  Shapes are those of the layers the
benchmark and tests use (16 or 32 query heads over 8 kv heads, head_dim 128 or 64, caches
of 1K to 32K rows, 1 to 64 streams) and generic odd ones.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rotary(name, batch, tokens, hq, hkv, d, rot, dtype, layout="half", scaling="none", start=0, ragged=False,
            train=False):
    case = {"op": "rotary", "batch": batch, "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "rot": rot,
            "dtype": dtype, "layout": layout, "scaling": scaling, "start": start, "ragged": ragged, "train": train}
    return {"name": name, **case} if name else case


def _append(name, batch, tokens, hq, hkv, d, rot, dtype, page, max_len, layout="half", scaling="none", ragged=False,
            idle=0):
    case = {"op": "append", "batch": batch, "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "rot": rot,
            "dtype": dtype, "page": page, "max_len": max_len, "layout": layout, "scaling": scaling,
            "ragged": ragged, "idle": idle}
    return {"name": name, **case} if name else case


def _attend(name, batch, hq, hkv, d, dtype, page, shared, own_min, own_max, idle=0):
    case = {"op": "attend", "batch": batch, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype, "page": page,
            "shared": shared, "own_min": own_min, "own_max": own_max, "idle": idle}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one stream's next token at the end of a 32K context: a launch, no bytes to speak of
        _rotary("rotary decode 1x1", 1, 1, 16, 8, 128, 128, "bf16", start=32767),
        # prefill of four 8K prompts, 32 query heads of 64 dims, llama3-scaled frequencies
        _rotary("rotary prefill 4x8192", 4, 8192, 32, 8, 64, 64, "bf16", scaling="llama3"),
        # a training step of the rotation, forward and backward
        _rotary("rotary train 8x2048", 8, 2048, 16, 8, 128, 128, "bf16", train=True),
        # interleaved pairs over half of an odd head, yarn-scaled, each sequence at its own far position, fp32
        _rotary("rotary yarn fp32 3x1021", 3, 1021, 12, 4, 96, 48, "fp32", layout="interleaved", scaling="yarn",
                start=1 << 20, ragged=True),
        # one stream's decode step into 16-row pages
        _append("append decode 1x1", 1, 1, 16, 8, 128, 128, "bf16", 16, 4096),
        # a 64-stream decode step into 64-row pages, a few batch rows idle as in a padded captured batch
        _append("append decode 64x1", 64, 1, 16, 8, 128, 128, "bf16", 64, 32768, idle=3),
        # ragged prefill of eight prompts of up to 4K tokens
        _append("append prefill 8x4096", 8, 4096, 32, 8, 64, 64, "bf16", 64, 8192, scaling="llama3", ragged=True),
        # interleaved, two thirds of the head, fp16, odd chunk lengths
        _append("append chunk fp16 5x333", 5, 333, 12, 4, 96, 64, "fp16", 32, 2048, layout="interleaved", ragged=True),
        # two streams just past a 1K prompt: latency
        _attend("attend 2 shared 1024", 2, 16, 8, 128, "bf16", 16, 1024, 1, 32),
        # 64 streams on a 4K prompt, own parts of up to a 1K window
        _attend("attend 64 shared 4096", 64, 16, 8, 128, "bf16", 64, 4096, 16, 1020, idle=3),
        # 256 streams on a 32K prompt, 64-dim heads, fp16: the shared part is a large matrix product
        _attend("attend 256 shared 32768", 256, 32, 8, 64, "fp16", 128, 32768, 64, 2048),
        # 64 streams with nothing shared, up to 16K rows each: every row read for one stream alone
        _attend("attend 64 own 16384", 64, 16, 8, 128, "bf16", 64, 0, 1024, 16384),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend"])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 7, 8])
    layout, scaling = rng.choice(["half", "interleaved"]), rng.choice(["none", "linear", "llama3", "yarn"])
    if op != "attend":
        d = rng.choice([40, 64, 80, 96, 112, 128, 256])
        rot = rng.choice([d, d, d // 2, max(2, d // 4 // 2 * 2)])
        batch = _log_int(rng, 1, 64)
        most = 4 * 8192 * 40 * 64 // (batch * (hq + hkv) * d)  # no more values than the largest listed case
        tokens = _log_int(rng, 1, max(1, min(8192, most)))
        if op == "rotary":
            train = rng.random() < 0.4
            return _rotary("", batch, tokens // 2 + 1 if train else tokens, hq, hkv, d, rot,
                           rng.choice(["bf16", "fp16", "bf16", "fp32"]) if tokens < most // 2 else "bf16", layout,
                           scaling, rng.choice([0, 31, 30000, 1 << 20]), rng.random() < 0.5, train)
        tokens = min(tokens, 4096, max(1, most // 2))
        return _append("", batch, tokens, hq, hkv, d, rot, rng.choice(["bf16", "fp16"]), rng.choice([16, 32, 64, 128]),
                       tokens + _log_int(rng, 1, 4096), layout, scaling, rng.random() < 0.6,
                       rng.choice([0, 0, 1]) if batch > 1 else 0)
    page, d = rng.choice([16, 32, 64, 128]), rng.choice([64, 128])
    batch = _log_int(rng, 1, 256)
    shared = rng.choice([0, 1]) * page * max(1, _log_int(rng, 64, 32768) // page)
    own_max = _log_int(rng, 1, max(1, min(16384, 64 * 8192 // batch)))
    if batch * hq * (shared + own_max) * 2 > 256 * 32 * 34816:
        shared = 1024
    return _attend("", batch, hq, hkv, d, rng.choice(["bf16", "fp16"]), page, shared,
                   _log_int(rng, 1, own_max), own_max, rng.choice([0, 0, 1]) if batch > 1 else 0)


# ------------------------------------------------------------------------------- inputs


def _spread(lo, hi, n, idle=0):
    """n whole numbers over [lo, hi], the last `idle` of them 0: the same for every seed, so
    that a case's work does not depend on it."""
    got = [lo + int((hi - lo) * ((i * 0.6180339887) % 1.0) + 0.5) for i in range(n)]
    return [hi if i == 0 else x for i, x in enumerate(got)][: n - idle] + [0] * idle


def _frequencies(rot, scaling):
    """(64-bit inverse frequencies, attention scaling) as a model's configuration gives them."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    if scaling == "llama3":
        f = 500000.0 ** (-i / rot)
        turns = 8192 * f / (2 * math.pi)  # turns over the original context: 1 and 4 are the borders
        mix = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - mix) * f / 32.0 + mix * f, 1.0
    f = 10000.0 ** (-i / rot)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "yarn":
        ramp = (torch.arange(rot // 2, dtype=torch.float64) / max(1, rot // 2 - 1)).clamp(0, 1)
        return f * (1 - ramp) + f / 16.0 * ramp, 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _lens_counts(case):
    """Cache lengths after the append, and how many of them are new, per sequence."""
    b, n = case["batch"], case["tokens"]
    live = b - case["idle"]
    counts = _spread(1 if case["ragged"] else n, n, live) + [0] * case["idle"]
    before = _spread(0, case["max_len"] - n, live)[::-1] + [0] * case["idle"]
    return [x + y for x, y in zip(before, counts)], counts


def _pages(case, lens, shared, gen):
    """(block table, number of pages): the shared positions' pages are the same for every
    sequence, the others each sequence's own, in random order."""
    page, b = case["page"], len(lens)
    width = max(1, max(-(-n // page) for n in lens))
    ns = shared // page
    own_pages = torch.tensor([max(0, -(-n // page) - ns) for n in lens])
    used = ns + int(own_pages.sum())
    order = torch.randperm(used + 3, generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    table = torch.zeros(b, width, dtype=torch.int32, device="cuda")
    table[:, :ns] = order[:ns]
    table[:, ns:][(torch.arange(width - ns) < own_pages[:, None]).cuda()] = order[ns:used]
    return table, used + 3


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    b, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dt)

    state = {"case": case}
    if case["op"] in ("rotary", "append"):
        n = case["tokens"]
        # as projections give them: [batch, tokens, heads, d] in memory, seen as [batch, heads, tokens, d]
        state["q"], state["k"] = randn(b, n, hq, d).transpose(1, 2), randn(b, n, hkv, d).transpose(1, 2)
        f, state["attention_scaling"] = _frequencies(case["rot"], case["scaling"])
        state["inv_freq"] = f.cuda()
    if case["op"] == "rotary":
        pos = torch.arange(n, device="cuda") + case["start"]
        if case["ragged"]:
            pos = pos + torch.randint(0, 4096, (b, 1), generator=gen, device="cuda")
        state["positions"] = pos
        if case["train"]:
            state["q"].requires_grad_(True)
            state["k"].requires_grad_(True)
            state["dq"], state["dk"] = randn(b, hq, n, d), randn(b, hkv, n, d)
        return state
    if case["op"] == "append":
        lens, counts = _lens_counts(case)
        state["v"] = randn(b, n, hkv, d).transpose(1, 2)
        state["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
        shared = 0
    else:
        lens = [case["shared"] + x if x else 0 for x in _spread(case["own_min"], case["own_max"], b, case["idle"])]
        state["q"] = randn(b, 1, hq, d).transpose(1, 2) * 2  # scores spread over a few units
        shared = case["shared"]
    state["block_table"], pages = _pages(case, lens, shared, gen)
    state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    state["k_pages"], state["v_pages"] = randn(pages, hkv, case["page"], d), randn(pages, hkv, case["page"], d)
    if own:  # the handle a serving loop keeps over these buffers
        from attention_sinks_b200 import PagedKVCache
        state["cache"] = PagedKVCache(state["k_pages"], state["v_pages"], state["block_table"], state["lens"],
                                      inv_freq=state.get("inv_freq"),
                                      interleaved=case.get("layout") == "interleaved",
                                      attention_scaling=state.get("attention_scaling", 1.0))
    return state


# ---------------------------------------------------------------------------- plain forms


def _cos_sin(positions, inv_freq, scaling):
    angles = positions[..., None].double() * inv_freq
    return (angles.cos() * scaling).float(), (angles.sin() * scaling).float()


def _turn(x, cos, sin, interleaved):
    """x [..., tokens, d] with its first 2 * cos.shape[-1] dims rotated, in 32 bits, rounded once."""
    r = 2 * cos.shape[-1]
    y = x.float()
    if interleaved:
        x1, x2 = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack((x1 * cos - x2 * sin, x2 * cos + x1 * sin), dim=-1).flatten(-2)
    else:
        x1, x2 = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), dim=-1)
    return torch.cat((turned, y[..., r:]), dim=-1).to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    pos = s["positions"] if s["positions"].dim() == 2 else s["positions"][None]
    cos, sin = _cos_sin(pos[:, None], s["inv_freq"], s["attention_scaling"])
    q = _turn(s["q"], cos, sin, case["layout"] == "interleaved")
    k = _turn(s["k"], cos, sin, case["layout"] == "interleaved")
    return q, k


def _plain_append(s):
    case = s["case"]
    page, n = case["page"], case["tokens"]
    t = torch.arange(n, device="cuda")
    pos = s["lens"].long()[:, None] - s["counts"].long()[:, None] + t
    live = t < s["counts"][:, None]
    cos, sin = _cos_sin(pos[:, None], s["inv_freq"], s["attention_scaling"])
    turned = _turn(s["k"], cos, sin, case["layout"] == "interleaved")
    q = _turn(s["q"], cos, sin, case["layout"] == "interleaved")
    bi, ti = live.nonzero(as_tuple=True)
    at = pos[bi, ti]
    row = s["block_table"][bi, at // page].long()
    s["k_pages"][row, :, at % page] = turned[bi, :, ti]
    s["v_pages"][row, :, at % page] = s["v"][bi, :, ti]
    q = torch.where(live[:, None, :, None], q, torch.zeros((), dtype=q.dtype, device="cuda"))
    return q, s["k_pages"], s["v_pages"]


def _plain_attend(s):
    case = s["case"]
    b, hq, hkv, d, page = case["batch"], case["hq"], case["hkv"], case["d"], case["page"]
    g, ns = hq // hkv, case["shared"] // case["page"]
    q = s["q"].float().reshape(b, hkv, g, d) * d ** -0.5
    own_table = s["block_table"][:, ns:].long()
    lens, width = s["lens"].long(), own_table.shape[1] * page

    def rows(pages, table):  # the table's pages as [..., hkv, rows, d]
        x = pages[table].float().transpose(-4, -3)
        return x.reshape(*x.shape[:-3], -1, d)

    j = torch.arange(width, device="cuda")
    seen = j < (lens - case["shared"])[:, None]
    scores = torch.matmul(q, rows(s["k_pages"], own_table).transpose(-1, -2))
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    if ns:
        first = s["block_table"][0, :ns].long()
        flat = q.transpose(0, 1).reshape(hkv, b * g, d)
        head = torch.matmul(flat, rows(s["k_pages"], first).transpose(-1, -2))
        head = head.reshape(hkv, b, g, -1).transpose(0, 1)
        head = head.masked_fill((lens == 0)[:, None, None, None], float("-inf"))
        scores = torch.cat((head, scores), dim=-1)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = (scores - top).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    own_p = p[..., ns * page:].masked_fill(~seen[:, None, None], 0.0)
    values = rows(s["v_pages"], own_table)
    out = torch.matmul(own_p, values)
    if ns:
        flat = p[..., :ns * page].transpose(0, 1).reshape(hkv, b * g, ns * page)
        out = out + torch.matmul(flat, rows(s["v_pages"], first)).reshape(hkv, b, g, d).transpose(0, 1)
    return out.reshape(b, 1, hq, d).to(s["q"].dtype)


def run(state):
    case = state["case"]
    if case["op"] == "attend":
        if own:
            return state["cache"].attend(state["q"], shared_len=case["shared"])
        return _plain_attend(state)
    if case["op"] == "append":
        if own:
            q = state["cache"].append(state["k"], state["v"], q=state["q"], counts=state["counts"])
            return q, state["k_pages"], state["v_pages"]
        return _plain_append(state)
    if own:
        from attention_sinks_b200 import rotary
        q, k = rotary(state["q"], state["k"], state["positions"], state["inv_freq"],
                      interleaved=case["layout"] == "interleaved", attention_scaling=state["attention_scaling"])
    else:
        q, k = _plain_rotary(state)
    if not case["train"]:
        return q, k
    gq, gk = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))
    return q.detach(), k.detach(), gq, gk


# ---------------------------------------------------------------------- work and exact values


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "rotary":
        values = case["batch"] * case["tokens"] * (hq + hkv) * d
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * values * size, "flops": passes * 3 * values * case["rot"] // d}
    if case["op"] == "append":
        _, counts = _lens_counts(case)
        values = sum(counts) * (hq + 2 * hkv) * d
        return {"bytes": 2 * values * size, "flops": 3 * sum(counts) * (hq + hkv) * case["rot"]}
    own_rows = sum(_spread(case["own_min"], case["own_max"], case["batch"], case["idle"]))
    live = case["batch"] - case["idle"]
    return {"bytes": size * (2 * hkv * d * (case["shared"] + own_rows) + 2 * case["batch"] * hq * d),
            "flops": 4 * hq * d * (live * case["shared"] + own_rows)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        hkv, d = case["hkv"], case["d"]
        q = s["q"].double()[:, :, 0].reshape(case["batch"], hkv, -1, d)
        out = torch.zeros_like(q)
        for i, n in enumerate(s["lens"].tolist()):
            if n:
                table = s["block_table"][i, :-(-n // case["page"])].long()
                k, v = (x[table].transpose(0, 1).reshape(hkv, -1, d)[:, :n].double()
                        for x in (s["k_pages"], s["v_pages"]))
                out[i] = torch.softmax(q[i] @ k.transpose(1, 2) / math.sqrt(d), dim=-1) @ v
        return out.reshape(case["batch"], 1, -1, d)
    inv, a = s["inv_freq"], s["attention_scaling"]
    if case["op"] == "rotary":
        pos = s["positions"].expand(case["batch"], -1)
    else:
        pos = (s["lens"] - s["counts"]).long()[:, None] + torch.arange(case["tokens"], device="cuda")
    # each pair as one complex number, turned by multiplication with a * exp(i angle)
    unit = torch.polar(torch.full_like(pos, 1, dtype=torch.float64)[..., None] * a,
                       pos.double()[..., None] * inv)[:, None]

    def turn(x, unit):
        r, y = case["rot"], x.detach().double().clone()
        first, second = (slice(0, r, 2), slice(1, r, 2)) if case["layout"] == "interleaved" else \
                        (slice(0, r // 2), slice(r // 2, r))
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * unit
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = turn(s["q"], unit), turn(s["k"], unit)
    if case["op"] == "rotary":
        if not case["train"]:
            return q, k
        return q, k, turn(s["dq"], unit.conj()), turn(s["dk"], unit.conj())
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    for i, count in enumerate(s["counts"].tolist()):
        q[i, :, count:] = 0
        at = pos[i, :count]
        row = s["block_table"][i].long()[at // case["page"]]
        kp[row, :, at % case["page"]] = k[i, :, :count].transpose(0, 1)
        vp[row, :, at % case["page"]] = s["v"][i, :, :count].double().transpose(0, 1)
    return q, kp, vp
