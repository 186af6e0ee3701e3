"""Operators of a serving step with a bounded attention window, as cases that can be timed and checked.

  decode   attention of one new query per sequence over a paged int4 / int8 cache, limited to the last `window`
           tokens and the first `sinks` ones (Ops.decode)
  prefill  the same limit on a prompt, or on a chunk over its history, in bf16 / fp16 rows: one length for the
           batch, or ragged rows packed end to end (window_attention)
  table    a decode step's block table, from an engine's token map and the requests' lengths (block_table)
  maps     a prefill step's index arrays from the requests' lengths: row offsets, pages to write, pages to unpack,
           rows and slots of the new tokens (step_maps)
  sample   one token per row from its logits and a given random number, with temperature, top-k, top-p and
           min-p (sample)

Query t of a sequence sees key j <= t when j > t - window or j < sinks.
"""
import math
import random

import torch

own = False

PAGE = 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one user's chat with a short window: launch and latency
        dict(name="decode_one", kind="decode", batch=1, tokens=1000, spread=0.0, empty=0, window=512, sinks=4, hkv=8,
             group=4, dim=128, bits=4, dtype="bf16"),
        # a busy server's long conversations: 64 sequences of up to 32,768 tokens, 28 q heads over 4 kv heads
        dict(name="decode_batch", kind="decode", batch=64, tokens=32768, spread=0.4, empty=0, window=4096, sinks=4,
             hkv=4, group=7, dim=128, bits=4, dtype="bf16"),
        # ragged lengths around a window that some do not fill, int8, narrow heads, a padded row
        dict(name="decode_ragged", kind="decode", batch=97, tokens=5000, spread=0.97, empty=1, window=1111, sinks=0,
             hkv=12, group=2, dim=64, bits=8, dtype="fp16"),
        # a short prompt
        dict(name="prompt_short", kind="prefill", batch=1, tokens=150, history=0, spread=0.0, packed=False, window=64,
             sinks=2, hkv=4, group=7, dim=64, dtype="bf16"),
        # a long prompt, four windows of sinks and neighbours deep
        dict(name="prompt_long", kind="prefill", batch=1, tokens=8192, history=0, spread=0.0, packed=False,
             window=2048, sinks=4, hkv=8, group=4, dim=128, dtype="bf16"),
        # follow-up turns of 9 conversations over their unpacked history
        dict(name="turns_packed", kind="prefill", batch=9, tokens=400, history=8000, spread=0.9, packed=True,
             window=1500, sinks=40, hkv=8, group=4, dim=128, dtype="fp16"),
        # a small decode batch's table
        dict(name="table_small", kind="table", batch=5, context=2048, tokens=700, spread=0.9),
        # a full server's table: 256 requests of up to 32,768 tokens
        dict(name="table_full", kind="table", batch=256, context=32768, tokens=32768, spread=0.95),
        # one chunk's maps
        dict(name="maps_chunk", kind="maps", batch=3, tokens=300, history=2000, spread=0.9, window=0, sinks=0),
        # a large prefill step: 64 requests with long histories, unpacked for a window
        dict(name="maps_step", kind="maps", batch=64, tokens=1024, history=32768, spread=0.9, window=8192, sinks=4),
        # a single user's next token over a large vocabulary, every filter on
        dict(name="sample_one", kind="sample", batch=1, vocab=152064, temperature=0.8, top_k=50, top_p=0.9,
             min_p=0.02, per_row=False, banned=0.0, dtype="bf16"),
        # a server's batch, each request with its own settings, some tokens masked
        dict(name="sample_batch", kind="sample", batch=64, vocab=151936, temperature=0.9, top_k=400, top_p=0.95,
             min_p=0.0, per_row=True, banned=0.1, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prefill", "prefill", "table", "maps", "sample", "sample"])
    heads = dict(hkv=rng.choice([1, 2, 4, 8, 12]), group=rng.choice([1, 2, 4, 7, 8, 12, 16]),
                 dim=rng.choice([64, 128, 128, 256]), dtype=rng.choice(["bf16", "fp16"]))
    window = dict(window=_log(rng, 1, 8192), sinks=rng.choice([0, 1, 4, rng.randint(2, 160)]))
    if kind == "decode":
        c = dict(kind=kind, batch=_log(rng, 1, 128), tokens=_log(rng, 1, 32768), spread=rng.choice([0.0, 0.5, 0.97]),
                 empty=rng.choice([0, 0, 1]), bits=rng.choice([4, 4, 8]), **window, **heads)
        # at most a third of the largest listed case's visible tokens and cached ones
        while c["batch"] * min(c["tokens"], c["window"] + c["sinks"]) * c["hkv"] * c["dim"] > 64 * 4100 * 512 // 3:
            c["batch"] = max(1, c["batch"] // 2)
            c["window"] = max(1, c["window"] * 3 // 4)
        while c["batch"] * c["tokens"] * c["hkv"] * c["dim"] > 64 * 32768 * 512 // 3:
            c["tokens"] = c["tokens"] // 2
        return c
    if kind == "prefill":
        c = dict(kind=kind, batch=_log(rng, 1, 12), tokens=_log(rng, 2, 4096),
                 history=rng.choice([0, _log(rng, 1, 12000)]), spread=rng.choice([0.0, 0.9]), packed=rng.random() < 0.5,
                 **window, **heads)
        if not c["packed"]:
            c["spread"] = 0.0
        c["hkv"] = min(c["hkv"], max(1, 32 // c["group"]))
        # score matrices of at most a third of the largest listed case's
        while (c["batch"] * c["hkv"] * c["group"] * c["tokens"] * (c["tokens"] + c["history"]) * c["dim"]
               > 32 * 8192 ** 2 * 128 // 3):
            c["tokens"], c["history"] = max(2, c["tokens"] * 2 // 3), c["history"] * 2 // 3
            c["batch"] = max(1, c["batch"] - 1)
        return c
    if kind == "table":
        tokens = _log(rng, 1, 32768)
        return dict(kind=kind, batch=_log(rng, 1, 200), context=_log(rng, tokens, 32768), tokens=tokens,
                    spread=rng.choice([0.0, 0.95]))
    if kind == "maps":
        return dict(kind=kind, batch=_log(rng, 1, 60), tokens=_log(rng, 1, 1000), history=rng.choice([0, _log(rng, 1, 32000)]),
                    spread=rng.choice([0.0, 0.9]), window=rng.choice([0, window["window"]]), sinks=window["sinks"])
    vocab = _log(rng, 100, 151000)
    return dict(kind=kind, batch=_log(rng, 1, 60), vocab=vocab, temperature=round(rng.uniform(0.3, 1.6), 3),
                top_k=rng.choice([0, _log(rng, 1, 5000)]), top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                min_p=rng.choice([0.0, round(10 ** rng.uniform(-4, -1), 5)]), per_row=rng.random() < 0.5,
                banned=rng.choice([0.0, 0.3]), dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))


# ------------------------------------------------------------------ sizes of a case
def _lengths(c, which, seed=None):
    """The sequences' lengths, between (1 - spread) and 1 times c[which], at least 1 where that is. They are the case's
    own, so that outputs have one size; a seed puts the sequences in an order of its own."""
    rng, most = random.Random("%s %s" % (which, sorted((k, v) for k, v in c.items() if k != "name"))), c[which]
    lens = [max(min(most, 1), int(most * (1 - rng.random() * c["spread"]))) for _ in range(c["batch"])]
    lens[:c.get("empty", 0)] = [0] * min(c.get("empty", 0), len(lens))
    if seed is not None:
        random.Random(seed).shuffle(lens)
    return lens


def _gap(first, c):
    """Pages that the window of the query at position `first` hides between the sinks' pages and its own."""
    return max(0, max(0, first - c["window"] + 1) // PAGE - -(-c["sinks"] // PAGE)) if c["window"] else 0


def _pairs(T, N, c):
    """Visible (query, key) pairs of T queries at the end of N keys."""
    t = torch.arange(N - T, N, dtype=torch.float64)
    near = torch.clamp(t + 1, max=c["window"])
    return float((near + torch.clamp(torch.clamp(t + 1 - near, max=c["sinks"]), min=0)).sum())


def work(c):
    D = c.get("dim", 0)
    if c["kind"] == "decode":
        lens = _lengths(c, "tokens")
        row = D if c["bits"] == 8 else D // 2
        see = sum(min(n, c["window"]) + min(c["sinks"], max(0, n - c["window"])) for n in lens)
        pages = sum(-(-n // PAGE) - _gap(n - 1, c) for n in lens if n)
        hq = c["hkv"] * c["group"]
        return {"bytes": c["hkv"] * (see * (2 * row + 4) + pages * 4 * D) + 4 * pages + 4 * c["batch"] * hq * D,
                "flops": 4.0 * see * hq * D}
    if c["kind"] == "prefill":
        T, H = _lengths(c, "tokens"), _lengths(c, "history")
        hq = c["hkv"] * c["group"]
        keys = sum(t + min(h, c["window"] - 1 + c["sinks"]) for t, h in zip(T, H))
        return {"bytes": 2 * D * (2 * sum(T) * hq + 2 * keys * c["hkv"]),
                "flops": 4.0 * D * hq * sum(_pairs(t, t + h, c) for t, h in zip(T, H))}
    if c["kind"] == "table":
        pages = sum(-(-n // PAGE) for n in _lengths(c, "tokens"))
        return {"bytes": 4 * pages + c["batch"] * (4 * -(-c["context"] // PAGE) + 24), "flops": pages}
    if c["kind"] == "maps":
        n = _map_sizes(_lengths(c, "tokens"), _lengths(c, "history"), c)
        return {"bytes": 12 * n["pages"] + 12 * n["jobs"] + 12 * n["tokens"] + 20 * n["tails"] + 24 * c["batch"],
                "flops": n["pages"] + n["jobs"] + n["tokens"]}
    size = {"fp32": 4}.get(c["dtype"], 2)
    return {"bytes": c["batch"] * (c["vocab"] * size + 12), "flops": 4 * c["batch"] * c["vocab"]}


def _map_sizes(T, H, c):
    return {"tokens": sum(T), "pages": sum(h // PAGE - _gap(h, c) for h in H), "tails": sum(h % PAGE > 0 for h in H),
            "jobs": sum((h + t - 1) // PAGE - h // PAGE + 1 for t, h in zip(T, H) if t)}


# ------------------------------------------------------------------ inputs
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _pages_of(lens, g, spare=0):
    """A block table over blocks in random order, and how many blocks there are."""
    pages = [-(-n // PAGE) for n in lens]
    total, wide = sum(pages) + 3, max(max(pages) + spare, 1)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    at = torch.arange(wide, device="cuda")[None, :]
    count = _ints(pages, torch.int64)[:, None]
    ids = order[(torch.cumsum(count, 0) - count + at).clamp(max=total - 1)]
    return torch.where(at < count, ids, torch.zeros_like(ids)).contiguous(), total


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = PREPARE[c["kind"]](c, seed, g)
    if own:
        import kushkash_amd as kk
        s["kk"] = kk
        if c["kind"] == "decode":                    # what a server keeps: the kernels' handle, the split count, its scratch
            ops = s["ops"] = kk.Ops(torch.device("cuda"), c["dim"], c["bits"], c["group"], s["q"].dtype)
            s["splits"] = ops.splits(c["batch"], c["hkv"], max(s["lens"]) // PAGE, window=c["window"], sinks=c["sinks"])
            s["work"] = torch.empty(c["batch"] * c["hkv"] * s["splits"] * c["group"] * (c["dim"] + 2),
                                    dtype=torch.float32, device="cuda")
    return s


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _prepare_decode(c, seed, g):
    D, H, B, dt = c["dim"], c["hkv"], c["batch"], DTYPES[c["dtype"]]
    lens = _lengths(c, "tokens", seed)
    table, blocks = _pages_of(lens, g)
    # records: codes of every value, scales that give unit spread, biases N(0, 1) that a tenth of the channels has six
    # times as large, nearly the same on every page (as keys have)
    body = 2 * PAGE * (D if c["bits"] == 8 else D // 2)
    step = 1.0 / (4.6 if c["bits"] == 4 else 74.0)
    records = torch.randint(0, 256, (blocks, H, body + 4 * D + 4 * PAGE), generator=g, device="cuda", dtype=torch.uint8)
    meta = torch.empty(blocks, H, 2 * D + 2 * PAGE, dtype=torch.float16, device="cuda")
    channel = torch.randn(H, D, generator=g, device="cuda")
    channel *= torch.where(torch.rand(H, D, generator=g, device="cuda") < 0.1, 6.0, 0.3)
    meta[..., :D] = step * (0.7 + 0.6 * torch.rand(blocks, H, D, generator=g, device="cuda"))
    meta[..., D:2 * D] = channel + 0.2 * torch.randn(blocks, H, D, generator=g, device="cuda")
    meta[..., 2 * D:2 * D + PAGE] = step * (0.7 + 0.6 * torch.rand(blocks, H, PAGE, generator=g, device="cuda"))
    meta[..., 2 * D + PAGE:] = 0.2 * torch.randn(blocks, H, PAGE, generator=g, device="cuda")
    records[..., body:] = meta.view(torch.uint8)
    tail = (channel[None, :, None] + _normal((B, H, PAGE, D), g, torch.float32)).to(dt)
    return dict(case=c, lens=lens, records=records, table=table, tail=tail, slots=torch.randperm(B, generator=g, device="cuda").to(torch.int32),
                seq_lens=_ints(lens), q=_normal((B, H * c["group"], D), g, dt),
                out=torch.empty(B, H * c["group"], D, dtype=dt, device="cuda"), scale=D ** -0.5)


def _prepare_prefill(c, seed, g):
    D, H, dt = c["dim"], c["hkv"], DTYPES[c["dtype"]]
    T, P = _lengths(c, "tokens", seed), _lengths(c, "history", seed)
    if not c["packed"]:
        T, P = [c["tokens"]] * c["batch"], [c["history"]] * c["batch"]
    N = [t + p for t, p in zip(T, P)]
    rows = (sum(T), sum(N)) if c["packed"] else ((c["batch"], T[0]), (c["batch"], N[0]))
    shape = [(n,) if c["packed"] else n for n in rows]
    starts = [_ints([0] + torch.tensor(x).cumsum(0).tolist()) for x in (T, N)]
    return dict(case=c, T=T, N=N, starts=starts, scale=D ** -0.5, q=_normal((*shape[0], H * c["group"], D), g, dt),
                k=_normal((*shape[1], H, D), g, dt), v=_normal((*shape[1], H, D), g, dt))


def _prepare_table(c, seed, g):
    lens = _lengths(c, "tokens", seed)
    rows = c["batch"] + 7
    blocks = torch.randint(1, 1 << 20, (rows, -(-c["context"] // PAGE)), generator=g, device="cuda", dtype=torch.int32)
    tokens = (blocks[:, :, None] * PAGE + torch.arange(PAGE, device="cuda", dtype=torch.int32)).view(rows, -1)
    return dict(case=c, req_to_token=tokens[:, :c["context"]].contiguous(), seq_lens=_ints(lens, torch.int64),
                req=torch.randperm(rows, generator=g, device="cuda")[:c["batch"]], pages=blocks.shape[1])


def _prepare_maps(c, seed, g):
    T, H = _lengths(c, "tokens", seed), _lengths(c, "history", seed)
    table, _ = _pages_of([t + h for t, h in zip(T, H)], g, spare=5)
    limit = dict(window=c["window"] or None, sinks=c["sinks"] if c["window"] else 0)
    return dict(case=c, T=T, H=H, limit=limit, new=_ints(T), history=_ints(H), table=table,
                slots=torch.randperm(c["batch"] + 9, generator=g, device="cuda")[:c["batch"]].to(torch.int32))


def _prepare_sample(c, seed, g):
    B, V = c["batch"], c["vocab"]
    x = 2.0 * torch.randn(B, V, generator=g, device="cuda") + 6.0 * torch.rand(B, V, generator=g, device="cuda") ** 12
    if c["banned"]:
        banned = torch.rand(B, V, generator=g, device="cuda") < c["banned"]
        banned[:, 0] = False
        x = torch.where(banned, float("-inf"), x)
    s = dict(case=c, logits=x.to(DTYPES[c["dtype"]]), u=torch.rand(B, generator=g, device="cuda"))
    for name, dtype in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32)):
        s[name] = c[name]
        if c["per_row"]:
            near = 0.6 + 0.4 * torch.rand(B, generator=g, device="cuda")
            s[name] = torch.where(near > 0.95, float(c[name]), c[name] * near).to(dtype)
    return s


PREPARE = dict(decode=_prepare_decode, prefill=_prepare_prefill, table=_prepare_table, maps=_prepare_maps,
               sample=_prepare_sample)


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if own:
        kk = s["kk"]
        if c["kind"] == "decode":
            s["ops"].decode(s["q"], s["out"], s["records"], s["table"], s["seq_lens"], s["slots"], s["tail"], s["scale"],
                            s["splits"], s["work"], window=c["window"], sinks=c["sinks"])
            return s["out"]
        if c["kind"] == "prefill":
            rows = dict(cu=(s["starts"][0], s["starts"][1]), spans=list(zip(s["T"], s["N"]))) if c["packed"] else {}
            return kk.window_attention(s["q"], s["k"], s["v"], window=c["window"], sinks=c["sinks"], scale=s["scale"], **rows)
        if c["kind"] == "table":
            return kk.block_table(s["req_to_token"], s["req"], s["seq_lens"], s["pages"])
        if c["kind"] == "maps":
            # (the lengths are another step's every time, so their sizes are part of the pass, as in the plain form)
            m = kk.step_maps(s["new"], s["history"], s["slots"], s["table"], kk.map_sizes(s["T"], s["H"], **s["limit"]))
            return [getattr(m, name) for name in MAPS]
        return kk.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return PLAIN[c["kind"]](s, c)


def _dequantized(rec, D, bits):
    """Records [..., RB] -> K, V [..., 32, D] fp32."""
    row = D if bits == 8 else D // 2
    codes = rec[..., :2 * PAGE * row].view(torch.int8).unflatten(-1, (2, PAGE, row))
    if bits == 4:
        codes = torch.cat([((codes & 15) ^ 8) - 8, codes >> 4], -1)
    par = rec[..., 2 * PAGE * row:].contiguous().view(torch.float16).float()
    K = codes[..., 0, :, :] * par[..., None, :D] + par[..., None, D:2 * D]
    V = codes[..., 1, :, :] * par[..., 2 * D:2 * D + PAGE, None] + par[..., 2 * D + PAGE:, None]
    return K, V


def _softmax_product(scores, hidden, V):
    """Rows of softmax(scores without what is hidden) V; a row that sees nothing is 0."""
    scores = scores.masked_fill_(hidden, float("-inf"))
    most = scores.amax(-1, keepdim=True)
    e = scores.sub_(torch.where(torch.isinf(most), torch.zeros_like(most), most)).exp_()
    total = e.sum(-1, keepdim=True)
    return (e @ V) / torch.where(total > 0, total, torch.ones_like(total))


def _plain_decode(s, c):
    D, H, B, W = c["dim"], c["hkv"], c["batch"], c["window"]
    n = s["seq_lens"].long()[:, None]
    count, first = (n + PAGE - 1) // PAGE, -(-c["sinks"] // PAGE)
    gap = ((n - W).clamp(min=0) // PAGE - first).clamp(min=0)
    p = torch.arange(min(s["table"].shape[1], first + (W + PAGE - 2) // PAGE + 1), device="cuda")[None, :]
    p = torch.where(p < first, p, p + gap)                                    # logical pages that are seen
    block = s["table"].long().gather(1, p.clamp(max=s["table"].shape[1] - 1))
    K, V = _dequantized(s["records"][block], D, c["bits"])                    # [B, pages, H, 32, D]
    part = ((p == count - 1) & (n % PAGE > 0))[:, :, None, None, None]
    K = torch.where(part, s["tail"].float()[s["slots"].long()][:, None], K)   # the last page's exact keys
    K, V = (x.transpose(1, 2).reshape(B, H, -1, D) for x in (K, V))
    at = (p[:, :, None] * PAGE + torch.arange(PAGE, device="cuda")).view(B, 1, 1, -1)
    m = n[:, :, None, None]
    hidden = (at >= m) | ((at < m - W) & (at >= c["sinks"]))
    q = s["q"].float().view(B, H, c["group"], D) * s["scale"]
    o = _softmax_product(q @ K.transpose(-1, -2).contiguous(), hidden, V.masked_fill_(hidden.transpose(-1, -2), 0.0))
    return o.reshape(s["q"].shape).to(s["q"].dtype)


def _plain_prefill(s, c):
    D, H, G, B = c["dim"], c["hkv"], c["group"], c["batch"]
    T, N = (_ints(x, torch.int64)[:, None] for x in (s["T"], s["N"]))
    t, j = (torch.arange(max(x), device="cuda")[None, :] for x in (s["T"], s["N"]))
    q, k, v = s["q"], s["k"], s["v"]
    if c["packed"]:                                                           # padded to the longest
        rows = (s["starts"][0][:-1, None] + t).clamp(max=q.shape[0] - 1)
        keys = (s["starts"][1][:-1, None] + j).clamp(max=k.shape[0] - 1)
        q, k, v = q[rows], k[keys], v[keys]
    q = (q.float() * s["scale"]).view(B, -1, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, D)
    k, v = (x.float().transpose(1, 2) for x in (k, v))
    at = (N - T + t)[:, :, None]                                              # the queries' positions
    hidden = (j[:, None] > at) | ((j[:, None] <= at - c["window"]) & (j[:, None] >= c["sinks"])) | (t >= T)[:, :, None]
    hidden = hidden[:, None].expand(B, G, -1, -1).reshape(B, 1, -1, j.shape[1])
    o = _softmax_product(q @ k.transpose(-1, -2).contiguous(), hidden, v.contiguous())
    o = o.view(B, H, G, -1, D).permute(0, 3, 1, 2, 4).reshape(B, -1, H * G, D)
    return (o[t < T] if c["packed"] else o).to(s["q"].dtype)


def _plain_table(s, c):
    pages = (s["seq_lens"] + PAGE - 1) // PAGE
    ids = s["req_to_token"][s["req"], ::PAGE] // PAGE
    seen = torch.arange(s["pages"], device="cuda")[None, :] < pages[:, None]
    return [torch.where(seen, ids, torch.zeros_like(ids)), s["seq_lens"].to(torch.int32), s["req"].to(torch.int32)]


MAPS = ("q_start", "key_start", "seq_lens", "job_seq", "job_page", "page_blk", "page_dst", "tail_blk", "tail_info",
        "new_dst", "slot_map")


def _runs(counts, total):
    """For runs of `counts` entries one behind the other: each entry's run, and its place in it."""
    run_of = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts, output_size=total)
    return run_of, torch.arange(total, device="cuda") - (torch.cumsum(counts, 0) - counts)[run_of]


def _plain_maps(s, c):
    T, H, table = s["new"].long(), s["history"].long(), s["table"]
    size = _map_sizes(s["T"], s["H"], c)
    first, full, gap = -(-c["sinks"] // PAGE), H // PAGE, torch.zeros_like(H)
    if c["window"]:
        gap = ((H - c["window"] + 1).clamp(min=0) // PAGE - first).clamp(min=0)
    kept = H - PAGE * gap
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    q_start, key_start = (torch.cat([zero, torch.cumsum(x, 0)]) for x in (T, kept + T))
    r, i = _runs(torch.where(T > 0, (H + T - 1) // PAGE - full + 1, T), size["jobs"])
    job_seq, job_page = r, full[r] + i
    r, i = _runs(full - gap, size["pages"])
    page_blk, page_dst = table[r, torch.where(i < first, i, i + gap[r])], key_start[r] + PAGE * i
    r, _ = _runs((H % PAGE > 0).long(), size["tails"])
    tail_blk = table[r, full[r]]
    tail_info = torch.stack([key_start[r] + PAGE * (full - gap)[r], H[r] % PAGE, s["slots"][r].long()], 1)
    r, i = _runs(T, size["tokens"])
    at = H[r] + i
    slot_map = table[r, at // PAGE].long() * PAGE + at % PAGE
    return [x.to(torch.int32) for x in (q_start, key_start, H + T, job_seq, job_page, page_blk, page_dst, tail_blk,
                                        tail_info, key_start[r] + kept[r] + i)] + [slot_map]


def _plain_sample(s, c):
    """In 64 bits: a token next to the border of what is kept, or of two tokens' shares, goes by the last digits."""
    B, V = s["logits"].shape
    T, k, p, m = (x.double()[:, None] if isinstance(x, torch.Tensor) else torch.full((B, 1), float(x), dtype=torch.float64, device="cuda")
                  for x in (s["temperature"], s["top_k"], s["top_p"], s["min_p"]))
    x, order = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / T)
    w = torch.where((k > 0) & (torch.arange(V, device="cuda") >= k), torch.zeros_like(w), w)
    before = torch.cumsum(w, -1) - w
    drop = ((p < 1) & (before >= p * w.sum(-1, keepdim=True))) | (w < m)
    drop[:, 0] = False
    w = torch.zeros_like(w).scatter_(1, order, w.masked_fill_(drop, 0.0))     # back in the vocabulary's order
    run = torch.cumsum(w, -1)
    return (run > s["u"].double()[:, None] * run[:, -1:]).int().argmax(-1)


PLAIN = dict(decode=_plain_decode, prefill=_plain_prefill, table=_plain_table, maps=_plain_maps, sample=_plain_sample)


# ------------------------------------------------------------------ the definition in 64 bits
def exact(c, seed):
    if c["kind"] not in ("decode", "prefill"):
        return None                                                           # whole numbers
    s = prepare(c, seed)
    G, W, scale = c["group"], c["window"], c["dim"] ** -0.5
    if c["kind"] == "decode":
        got = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"]):
            if not n:
                continue
            see = torch.tensor(sorted(set(range(min(n, c["sinks"]))) | set(range(max(0, n - W), n))), device="cuda")
            rec = s["records"][s["table"][b].long()[see // PAGE]]             # a record for each token
            K, V = _one_token(rec, see % PAGE, c)
            if n % PAGE:
                last = see >= n // PAGE * PAGE
                K[last] = s["tail"][int(s["slots"][b])][:, see[last] % PAGE].transpose(0, 1).double()
            for h in range(c["hkv"]):
                q = s["q"][b, h * G:(h + 1) * G].double()
                got[b, h * G:(h + 1) * G] = torch.softmax(scale * q @ K[:, h].T.contiguous(), -1) @ V[:, h]
        return got
    flat = [x.flatten(0, -3) for x in (s["q"], s["k"], s["v"])]
    got = torch.zeros(flat[0].shape, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for T, N in zip(s["T"], s["N"]):
        for a in range(0, T, 1024):                                           # queries a .. b - 1 and what they can see
            b = min(T, a + 1024)
            at = torch.arange(N - T + a, N - T + b, device="cuda")[:, None]
            low = max(0, N - T + a - W + 1)
            key = torch.tensor(list(range(min(c["sinks"], low))) + list(range(low, N - T + b)), device="cuda")
            bias = torch.where((key <= at) & ((key > at - W) | (key < c["sinks"])), 0.0, float("-inf")).double()
            for h in range(c["hkv"]):
                K, V = (x[k0 + key, h].double() for x in flat[1:])
                Kt = K.T.contiguous()
                for i in range(h * G, (h + 1) * G):
                    got[q0 + a:q0 + b, i] = torch.softmax(scale * flat[0][q0 + a:q0 + b, i].double() @ Kt + bias, -1) @ V
        q0, k0 = q0 + T, k0 + N
    return got.view(s["q"].shape)


def _one_token(rec, row, c):
    """Token row[i] of record rec[i] ([n, H, RB]), dequantized in 64 bits: K, V [n, H, D]."""
    D, int4 = c["dim"], c["bits"] == 4
    width = D // 2 if int4 else D
    i = torch.arange(len(row), device="cuda")
    half = rec[..., 2 * PAGE * width:].contiguous().view(torch.float16).double()
    out = []
    for part in (0, 1):
        code = rec[..., :2 * PAGE * width].unflatten(-1, (2 * PAGE, width))[i, :, part * PAGE + row].long()
        if int4:
            code = torch.cat([code % 16, code // 16], -1)
        code = torch.where(code >= (8 if int4 else 128), code - (16 if int4 else 256), code)
        sc, bi = ((half[..., :D], half[..., D:2 * D]) if part == 0 else
                  (half[i, :, 2 * D + row][..., None], half[i, :, 2 * D + PAGE + row][..., None]))
        out.append(code * sc + bi)
    return out
