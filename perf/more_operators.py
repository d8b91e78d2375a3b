"""The operators between a decoder's q/k/v and output projections, as cases that can be timed and compared.

Three of them: rotary positions (`rotary`), appending keys and values to a paged cache with the rotation applied on the way
(`paged_append`), and attention of a chunk of new tokens, one of them or many, over that cache (`paged_attention`).  A cache is a
pair of tensors (pages, page_size, kv_heads, head_dim); a sequence's keys lie in the pages that its row of the page table names.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
#: how frequencies are stretched for contexts longer than those a model was trained on
SCALINGS = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 4.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192},
    "yarn": {"rope_type": "yarn", "factor": 4.0, "beta_fast": 32.0, "beta_slow": 1.0, "original_max_position_embeddings": 32768},
}


# ------------------------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # queries and keys of one token of a small decoder (16 query and 4 key heads) in a decode step: latency alone
        dict(name="rotary_1x20x128", kind="rotary", tokens=1, heads=20, head_dim=128, rotary_dim=128, interleaved=False, base=5e6, scaling="none", first=4095, dtype="bf16"),
        # queries and keys (32 and 8 heads) of a long prompt, one token short of 8192, at far positions of a stretched context
        dict(name="rotary_8191x40x128_llama3", kind="rotary", tokens=8191, heads=40, head_dim=128, rotary_dim=128, interleaved=False, base=5e5, scaling="llama3", first=120000, dtype="bf16"),
        # one token's keys and values into the cache, its queries rotated in the same call: a decode step
        dict(name="append_1tok_16h4", kind="append", tokens=1, heads=16, kv_heads=4, head_dim=128, rotary_dim=128, interleaved=False, base=5e6, scaling="none", first=4095, pages=512,
             page_size=16, padding=0, dtype="bf16"),
        # a padded batch of 250 decoding sequences, neighbouring values paired, half of each head rotated
        dict(name="append_250tok_32h8_half", kind="append", tokens=256, heads=32, kv_heads=8, head_dim=128, rotary_dim=64, interleaved=True, base=1e4, scaling="yarn", first=90000, pages=1024,
             page_size=16, padding=6, dtype="fp16"),
        # a prompt of 4096 tokens
        dict(name="append_4096tok_32h16", kind="append", tokens=4096, heads=32, kv_heads=16, head_dim=128, rotary_dim=128, interleaved=False, base=1e6, scaling="linear", first=0, pages=512,
             page_size=16, padding=0, dtype="bf16"),
        # one sequence of 4096 tokens, one new one, small decoder: the smallest decode step
        dict(name="attend_1seq_4096_16h4", kind="attend", seqs=1, chunk=1, context=4095, ragged=False, heads=16, kv_heads=4, head_dim=128, page_size=16, window=0, dtype="bf16"),
        # 64 sequences of very different lengths, one new token each
        dict(name="attend_64seq_8192_32h8", kind="attend", seqs=64, chunk=1, context=8191, ragged=True, heads=32, kv_heads=8, head_dim=128, page_size=16, window=0, dtype="bf16"),
        # one token behind a very long context
        dict(name="attend_1seq_131072_32h8", kind="attend", seqs=1, chunk=1, context=131071, ragged=False, heads=32, kv_heads=8, head_dim=128, page_size=64, window=0, dtype="fp16"),
        # a whole prompt of 2048 tokens, wide dense decoder
        dict(name="attend_2048new_32h16", kind="attend", seqs=1, chunk=2048, context=0, ragged=False, heads=32, kv_heads=16, head_dim=128, page_size=16, window=0, dtype="bf16"),
        # a chunk of 512 tokens of a prompt, 16384 tokens already in the cache
        dict(name="attend_512new_16384_32h8", kind="attend", seqs=1, chunk=512, context=16384, ragged=False, heads=32, kv_heads=8, head_dim=128, page_size=32, window=0, dtype="bf16"),
        # a mixed batch: chunks of 1 to 333 tokens behind contexts of 0 to 5000, a sliding window, odd groups of heads
        dict(name="attend_24seq_mixed_15h3_window", kind="attend", seqs=24, chunk=333, context=5000, ragged=True, heads=15, kv_heads=3, head_dim=64, page_size=16, window=1024, dtype="fp16"),
        # a whole prompt of 8192 tokens
        dict(name="attend_8192new_32h8", kind="attend", seqs=1, chunk=8192, context=0, ragged=False, heads=32, kv_heads=8, head_dim=128, page_size=16, window=0, dtype="bf16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["rotary", "append", "attend", "attend", "attend", "attend"])
    if kind != "attend":
        head_dim = rng.choice([64, 128, 128, 8 * rng.randint(4, 16)])
        case = dict(kind=kind, head_dim=head_dim, rotary_dim=rng.choice([head_dim, head_dim // 4 * 2, 2 * rng.randint(1, head_dim // 2)]), interleaved=rng.random() < 0.5,
                    base=rng.choice([1e4, 5e5, 5e6]), scaling=rng.choice(sorted(SCALINGS)), first=rng.choice([0, log_int(1, 1000000)]))
        if kind == "rotary":
            return dict(case, tokens=log_int(1, 8191), heads=log_int(1, 40), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        kv_heads, page_size, tokens = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([16, 32, 64, 128]), log_int(1, 4096)
        return dict(case, tokens=tokens, heads=min(32, kv_heads * rng.choice([1, 2, 4, 5, 8])) // kv_heads * kv_heads, kv_heads=kv_heads, page_size=page_size,
                    pages=-(-tokens // page_size) + log_int(1, 256), padding=rng.choice([0, 0, rng.randint(0, tokens)]), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    while True:
        seqs = rng.choice([1, 1, rng.randint(2, 16), log_int(1, 128)])
        chunk = rng.choice([1, 1, rng.randint(2, 16), log_int(1, 8192)])
        context = rng.choice([0, log_int(1, 131071), log_int(1, 16384)])
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 8])
        case = dict(kind=kind, seqs=seqs, chunk=chunk, context=context, ragged=seqs > 1 and rng.random() < 0.7, heads=heads, kv_heads=kv_heads,
                    head_dim=rng.choice([64, 128, 128, 8 * rng.randint(4, 16)]), page_size=rng.choice([16, 16, 32, 64, 128]), window=rng.choice([0, 0, 0, log_int(16, 4096)]),
                    dtype=rng.choice(["bf16", "bf16", "fp16"]))
        if heads <= 32 and seqs * (chunk + context) * kv_heads * case["head_dim"] <= 64 * 8192 * 8 * 128 \
                and seqs * chunk * (chunk + context) * heads * case["head_dim"] <= 8192 * 8192 * 32 * 128:
            return case


def _sizes(case):
    """New tokens and keys of every sequence, from the case alone: a ragged one's spread over the range, the first one the longest."""
    new, keys = [], []
    for i in range(case["seqs"]):
        f, g = ((1.0 - i * 0.6180339887) % 1.0, (1.0 - i * 0.7548776662) % 1.0) if i and case["ragged"] else (1.0, 1.0)
        n = max(1, round(case["chunk"] * f))
        new.append(n)
        keys.append(n + round(case["context"] * g))
    return new, keys


def _seen(n, k, window):
    """Pairs of a query and a key that it sees: the n last of k positions, each up to its own, `window` of them at most."""
    first, most = k - n + 1, window or k                   # (query i sees min(first + i, most))
    short = max(0, min(n, most - first))
    return short * first + short * (short - 1) // 2 + (n - short) * most


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "attend":
        new, keys = _sizes(case)
        w, row = case["window"], case["head_dim"] * size
        kv = sum(min(k, w + n - 1) if w else k for n, k in zip(new, keys))
        pages = sum(-(-k // case["page_size"]) for k in keys)
        return {"bytes": 2 * sum(new) * case["heads"] * row + 2 * kv * case["kv_heads"] * row + 4 * pages + 8 * case["seqs"],
                "flops": 4 * case["heads"] * case["head_dim"] * sum(_seen(n, k, w) for n, k in zip(new, keys))}
    if case["kind"] == "rotary":
        values = case["tokens"] * case["heads"]
        return {"bytes": 2 * values * case["head_dim"] * size + 8 * case["tokens"], "flops": 3 * values * case["rotary_dim"]}
    used = case["tokens"] - case["padding"]
    return {"bytes": 2 * (case["tokens"] * case["heads"] + 2 * used * case["kv_heads"]) * case["head_dim"] * size + 16 * case["tokens"],
            "flops": 3 * (case["tokens"] * case["heads"] + used * case["kv_heads"]) * case["rotary_dim"]}


# ------------------------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------------------------
def _frequencies(dim, base, scaling, device):
    """(radians per position of every pair, in 64 bits; the factor on cosine and sine)."""
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    if scaling is None:
        return f, 1.0
    factor = scaling["factor"]
    if scaling["rope_type"] == "linear":
        return f / factor, 1.0
    old = scaling["original_max_position_embeddings"]
    if scaling["rope_type"] == "llama3":
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        keep = ((old * f / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return f * keep + f / factor * (1.0 - keep), 1.0
    # yarn: pairs that turn often enough within the old context stay, slow ones are stretched, with a ramp over the pairs between

    def pair(turns):
        return dim * math.log(old / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    lo, hi = max(math.floor(pair(scaling["beta_fast"])), 0), min(math.ceil(pair(scaling["beta_slow"])), dim - 1)
    ramp = ((torch.arange(dim // 2, dtype=torch.float64, device=device) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return f / factor * ramp + f * (1.0 - ramp), 0.1 * math.log(factor) + 1.0


def _rotated(x, positions, freq, scale, interleaved):
    """x (tokens, heads, head_dim) in 32 bits, the first 2 * len(freq) values of every head rotated."""
    pairs, x = freq.numel(), x.float()
    angle = positions.double()[:, None] * freq                     # (64 bits: positions are far)
    cos, sin = (torch.cos(angle) * scale).float()[:, None], (torch.sin(angle) * scale).float()[:, None]
    out = x.clone()
    a = x[..., 0:2 * pairs:2] if interleaved else x[..., :pairs]
    b = x[..., 1:2 * pairs:2] if interleaved else x[..., pairs:2 * pairs]
    u, v = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        out[..., 0:2 * pairs:2], out[..., 1:2 * pairs:2] = u, v
    else:
        out[..., :pairs], out[..., pairs:2 * pairs] = u, v
    return out


def _plain_append(s):
    rotate = lambda x: _rotated(x, s["positions"], s["freq"], s["factor"], s["interleaved"]).to(x.dtype)
    at = s["slots"][:s["used"]].long()                             # (the padding is behind)
    s["keys"].view(-1, *s["keys"].shape[2:])[at] = rotate(s["key"])[:s["used"]]
    s["values"].view(-1, *s["values"].shape[2:])[at] = s["value"][:s["used"]]
    return rotate(s["query"]), s["keys"], s["values"]


def _plain_attend(s):
    out = torch.empty_like(s["query"])
    heads, kv_heads = s["query"].shape[1], s["keys"].shape[2]
    group, scale, row = heads // kv_heads, s["query"].shape[2] ** -0.5, 0
    for i, (n, k) in enumerate(zip(s["new"], s["held"])):
        pages = s["pages"][i, :-(-k // s["keys"].shape[1])].long()
        keys, values = s["keys"][pages].flatten(0, 1)[:k], s["values"][pages].flatten(0, 1)[:k]
        at, key = torch.arange(k - n, k, device=out.device)[:, None], torch.arange(k, device=out.device)[None]
        hidden = key > at
        if s["window"]:
            hidden = hidden | (key <= at - s["window"])
        for h in range(kv_heads):
            q = s["query"][row:row + n, h * group:(h + 1) * group].transpose(0, 1).float()
            score = (q @ keys[:, h].float().t()) * scale
            score.masked_fill_(hidden, -math.inf)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            y = (p @ values[:, h].float()) / p.sum(-1, keepdim=True)
            out[row:row + n, h * group:(h + 1) * group] = y.transpose(0, 1).to(out.dtype)
        row += n
    return out


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _heads(g, rows, heads, head_dim, dtype):
    """Normal values with a few channels that stand out, as queries and keys have them."""
    x = torch.randn(rows, heads, head_dim, generator=g, device="cuda")
    x *= torch.where(torch.rand(heads, head_dim, generator=g, device="cuda") < 0.02, 3.0, 1.0)
    return x.to(DTYPES[dtype])


def _inputs(case, seed):
    g, kind, d, dtype = _gen(seed), case["kind"], case["head_dim"], case["dtype"]
    s = dict(kind=kind)
    if kind == "attend":
        new, held = _sizes(case)
        ps, kv = case["page_size"], case["kv_heads"]
        used = [-(-k // ps) for k in held]
        total = sum(used) + 3
        s["keys"] = _heads(g, total * ps, kv, d, dtype).view(total, ps, kv, d)
        s["values"] = torch.randn(total, ps, kv, d, generator=g, device="cuda").to(DTYPES[dtype])
        s["query"] = _heads(g, sum(new), case["heads"], d, dtype)
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)       # pages are handed out in any order
        pages, at = torch.zeros(case["seqs"], max(used), dtype=torch.int32, device="cuda"), 0
        for i, n in enumerate(used):
            pages[i, :n] = order[at:at + n]
            at += n
        offsets = [0]
        for n in new:
            offsets.append(offsets[-1] + n)
        s.update(pages=pages, lengths=torch.tensor(held, dtype=torch.int32, device="cuda"), offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"), new=new, held=held,
                 most=max(new), window=case["window"])
        return s
    t = case["tokens"]
    s["positions"] = torch.arange(case["first"], case["first"] + t, dtype=torch.int64, device="cuda")
    s["interleaved"] = case["interleaved"]
    if kind == "rotary":
        s["x"] = _heads(g, t, case["heads"], d, dtype)
        return s
    ps, kv = case["page_size"], case["kv_heads"]
    s["query"], s["key"] = _heads(g, t, case["heads"], d, dtype), _heads(g, t, kv, d, dtype)
    s["value"] = torch.randn(t, kv, d, generator=g, device="cuda").to(DTYPES[dtype])
    s["keys"], s["values"] = (torch.randn(case["pages"], ps, kv, d, generator=g, device="cuda").to(DTYPES[dtype]) for _ in range(2))
    s["used"] = t - case["padding"]
    # rows of whole pages in any order, as a prompt fills them; a batch of decoding sequences has its rows anywhere
    order = torch.randperm(case["pages"], generator=g, device="cuda")
    slots = (order[:, None] * ps + torch.arange(ps, device="cuda")).flatten()
    s["slots"] = (slots if t > 512 else slots[torch.randperm(slots.numel(), generator=g, device="cuda")])[:t].clone()
    s["slots"][s["used"]:] = -1
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if s["kind"] != "attend":
        # the frequencies as a program keeps them, made once for a model
        scaling = SCALINGS[case["scaling"]]
        if own:
            from glq_b200 import ops
            s["table"] = ops.rotary_table(case["rotary_dim"], base=case["base"], scaling=scaling, interleaved=case["interleaved"], device="cuda")
        else:
            s["freq"], s["factor"] = _frequencies(case["rotary_dim"], case["base"], scaling, "cuda")
    return s


def run(state):
    s = state
    if own:
        from glq_b200 import ops
        if s["kind"] == "rotary":
            return ops.rotary(s["x"], s["positions"], s["table"])
        if s["kind"] == "append":
            q = ops.paged_append(s["key"], s["value"], s["keys"], s["values"], s["slots"], positions=s["positions"], table=s["table"], query=s["query"])
            return q, s["keys"], s["values"]
        return ops.paged_attention(s["query"], s["keys"], s["values"], s["pages"], s["lengths"], query_offsets=s["offsets"], max_query_len=s["most"], window=s["window"])
    if s["kind"] == "rotary":
        return _rotated(s["x"], s["positions"], s["freq"], s["factor"], s["interleaved"]).to(s["x"].dtype)
    return _plain_append(s) if s["kind"] == "append" else _plain_attend(s)


# ------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, apart from the plain forms
# ------------------------------------------------------------------------------------------------------------------
def _exact_rotated(x, case, positions):
    """Pairs as complex numbers times e^(i angle)."""
    dim, base, scaling = case["rotary_dim"], case["base"], SCALINGS[case["scaling"]]
    freq, scale = [], 1.0
    kind = scaling["rope_type"] if scaling else None
    for i in range(dim // 2):
        f = math.exp(-2.0 * i / dim * math.log(base))
        if kind == "linear":
            f /= scaling["factor"]
        elif kind == "llama3":
            length, old = 2.0 * math.pi / f, scaling["original_max_position_embeddings"]
            if length > old / scaling["low_freq_factor"]:
                f /= scaling["factor"]
            elif length >= old / scaling["high_freq_factor"]:
                keep = (old / length - scaling["low_freq_factor"]) / (scaling["high_freq_factor"] - scaling["low_freq_factor"])
                f = (1.0 - keep) * f / scaling["factor"] + keep * f
        elif kind == "yarn":
            old, scale = scaling["original_max_position_embeddings"], 1.0 + math.log(scaling["factor"]) / 10.0
            where = [dim / 2.0 * math.log(old / (2.0 * math.pi * turns)) / math.log(base) for turns in (scaling["beta_fast"], scaling["beta_slow"])]
            lo, hi = max(0, math.floor(where[0])), min(dim - 1, math.ceil(where[1]))
            keep = 1.0 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = f * keep + (1.0 - keep) * f / scaling["factor"]
        freq.append(f)
    angle = positions.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.full_like(angle, scale), angle)
    x = x.double()
    part = x[..., :dim]
    if case["interleaved"]:
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], dim // 2, 2).contiguous()) * turn
        part = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(part[..., :dim // 2].contiguous(), part[..., dim // 2:].contiguous()) * turn
        part = torch.cat((z.real, z.imag), -1)
    return torch.cat((part, x[..., dim:]), -1)


def _exact_attend(s):
    query, table = s["query"].double(), s["pages"].tolist()
    ps, kv_heads = s["keys"].shape[1:3]
    group, out, row = query.shape[1] // kv_heads, torch.zeros_like(query), 0
    for i, (n, k) in enumerate(zip(s["new"], s["held"])):
        rows = torch.tensor(table[i], device=query.device).repeat_interleave(ps)[:k] * ps + torch.arange(k, device=query.device) % ps
        for h in range(kv_heads):
            keys, values = s["keys"][:, :, h].flatten(0, 1)[rows].double(), s["values"][:, :, h].flatten(0, 1)[rows].double()
            for a in range(0, n, 1024):
                b = min(n, a + 1024)
                where = torch.arange(k - n + a, k - n + b, device=query.device)
                back = where[:, None] - torch.arange(k, device=query.device)         # how far a key lies behind its query
                seen = (back >= 0) & (back < (s["window"] or k))
                z = torch.einsum("qgd,kd->gqk", query[row + a:row + b, h * group:(h + 1) * group], keys) / math.sqrt(query.shape[2])
                p = torch.softmax(torch.where(seen, z, -math.inf), -1)
                out[row + a:row + b, h * group:(h + 1) * group] = torch.einsum("gqk,kd->qgd", p, values)
        row += n
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if s["kind"] == "attend":
        return _exact_attend(s)
    if s["kind"] == "rotary":
        return _exact_rotated(s["x"], case, s["positions"])
    keys, values = s["keys"].double(), s["values"].double()
    rotated = _exact_rotated(s["key"], case, s["positions"])
    page, within = s["slots"][:s["used"]] // case["page_size"], s["slots"][:s["used"]] % case["page_size"]
    keys[page, within], values[page, within] = rotated[:s["used"]], s["value"][:s["used"]].double()
    return _exact_rotated(s["query"], case, s["positions"]), keys, values
