"""What is measured of the quantized key/value cache and the attention that reads it.

Three operators, as a GPT-OSS style engine calls them between its Q/K/V and its output
projection, at that model's heads (64 query heads on 8 key/value heads of 64, YaRN,
attention sinks, a window of 128 on every other layer) and at generic other ones:

  store   rotates the queries and keys of a batch's rows (YaRN) and writes keys and values
          into the paged cache in blocks of 32 (Q4_0 or Q8_0); then the rows are read back,
          so that the updated cache is seen as the values that it stands for.
  read    reads rows of the cache back as fp32 keys and values.
  attend  attention of a batch's rows over the cache: causal, grouped heads, an optional
          sliding window, an optional sink logit for each head.

A batch is `seqs` sequences, the longest `len` positions after its new rows, each with up
to `new` new rows (its last positions); "ragged": the others are shorter, by a rule of the
case alone.  Pages of `page` positions are dealt to the sequences in random order.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
ROPE = {"base": 150000.0, "factor": 32.0, "original": 4096, "fast": 32.0, "slow": 1.0}


def _case(name, kind, type, seqs, new, len, ragged=False, heads=64, kv=8, dim=64, page=128, window=0, sinks=True):
    return {"name": name, "kind": kind, "type": type, "seqs": seqs, "new": new, "len": len, "ragged": ragged,
            "heads": heads, "kv": kv, "dim": dim, "page": page, "window": window, "sinks": sinks}


def listed():
    return [
        # One sequence being generated: its new token enters the cache.
        _case("store_decode_1", "store", "q4_0", 1, 1, 1537),
        # A busy server's decode step, 8-bit cache, small pages.
        _case("store_decode_64", "store", "q8_0", 64, 1, 4097, ragged=True, page=32),
        # A long prompt enters the cache in one go.
        _case("store_prompt_4099", "store", "q4_0", 1, 4099, 4099),
        # A few short shared prefixes are taken out of the cache.
        _case("read_ragged_203", "read", "q8_0", 3, 203, 203, ragged=True, kv=4, heads=32, dim=128, page=64),
        # A whole long sequence is taken out (to move it to another engine).
        _case("read_16384", "read", "q4_0", 1, 16384, 16384),
        # Generation, a window layer of the model: latency counts.
        _case("decode_1_window", "attend", "q4_0", 1, 1, 1537, window=128),
        # Generation far into a long document, a full layer.
        _case("decode_1_long", "attend", "q4_0", 1, 1, 131071),
        # A busy server's decode step, full layer, sequences of all lengths.
        _case("decode_64_ragged", "attend", "q4_0", 64, 1, 8192, ragged=True),
        # The same with an 8-bit cache, heads of 128, no sinks, an odd group of heads.
        _case("decode_17_q8_dim128", "attend", "q8_0", 17, 1, 5003, ragged=True, heads=40, kv=8, dim=128, page=32, sinks=False),
        # A prompt's next chunk of 32 tokens over what is in the cache already.
        _case("chunk_32", "attend", "q4_0", 1, 32, 2049),
        # A prompt of 2,048 tokens at once, full layer.
        _case("prompt_2048", "attend", "q4_0", 1, 2048, 2048),
        # Several prompts of unequal lengths together, window layer, 8-bit cache.
        _case("prompts_ragged_window", "attend", "q8_0", 5, 1021, 1021, ragged=True, window=128, page=64),
    ]


def draw(rng):
    def span(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    most_flops = max(work(c)["flops"] for c in listed() if c["kind"] == "attend")
    most_bytes = {k: max(work(c)["bytes"] for c in listed() if c["kind"] == k) for k in ("store", "read", "attend")}
    kind = rng.choice(("store", "read", "attend", "attend", "attend"))
    while True:
        c = {"kind": kind, "type": rng.choice(("q4_0", "q8_0")), "dim": rng.choice((64, 64, 128)),
             "kv": rng.choice((1, 2, 4, 8)), "page": rng.choice((32, 64, 96, 128, 256)), "ragged": rng.random() < 0.6,
             "window": rng.choice((0, 0, 128, span(1, 1000))), "sinks": rng.random() < 0.6}
        c["heads"] = c["kv"] * rng.choice((1, 2, 3, 4, 5, 8, 8, 16))
        c["new"] = rng.choice((1, span(1, 16), span(1, 4096)))
        c["len"] = max(c["new"], span(1, 131072))
        c["seqs"] = span(1, 64) if c["new"] < 64 else span(1, 8)
        w = work(c)
        if w["flops"] <= most_flops and w["bytes"] <= most_bytes[kind] and c["seqs"] * c["len"] * c["kv"] * c["dim"] <= 1 << 28:
            return c


# ---- what a case's batch looks like, by the case alone

def _batch(c):
    """(new, len) of each sequence; the first has the case's own."""
    new, lens = [], []
    for i in range(c["seqs"]):
        f, g = (i * 0.6180339887 % 1.0, i * 0.7548776662 % 1.0) if c["ragged"] else (0.0, 0.0)
        n = max(1, c["new"] - int(0.75 * f * c["new"]))
        new.append(n)
        lens.append(max(n, c["len"] - int(0.75 * (f if c["len"] == c["new"] else g) * c["len"])))
    return new, lens


def _bits(c):
    return 4 if c["type"] == "q4_0" else 8


def _tile_bytes(c):
    """Bytes of 32 positions of one key/value head: codes and fp16 scales of the keys, then of the values."""
    return 2 * (32 * c["dim"] * _bits(c) // 8 + 32 * c["dim"] // 32 * 2)


def work(case):
    c = case
    new, lens = _batch(c)
    rows, kvd, qd = sum(new), c["kv"] * c["dim"], c["heads"] * c["dim"]
    stored = _tile_bytes(c) // 32 * c["kv"]  # one position, keys and values
    if c["kind"] == "read":
        return {"bytes": rows * (stored + 8 * kvd), "flops": 2 * rows * 2 * kvd}
    if c["kind"] == "store":
        # q read and written, k and v read, the cache written; the rows read back: the cache read, fp32 written
        return {"bytes": rows * (8 * qd + 8 * kvd + stored) + rows * (stored + 8 * kvd),
                "flops": rows * (3 * qd + 3 * kvd + 8 * kvd + 4 * kvd)}
    pairs = seen = 0
    for n, l in zip(new, lens):
        w = c["window"] or l
        first, last = l - n + 1, l  # positions that the first and the last new row see, without the window
        full = max(0, last - max(first, w) + 1)  # rows whose whole window is there
        part = n - full
        pairs += full * w + part * first + part * (part - 1) // 2
        seen += min(l, n + w - 1)
    return {"bytes": seen * stored + rows * 8 * qd + (c["heads"] * 4 if c["sinks"] else 0), "flops": 4 * c["dim"] * c["heads"] * pairs}


# ---- inputs

def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    new, lens = _batch(c)
    n_pages = [-(-l // c["page"]) for l in lens]
    order = torch.randperm(sum(n_pages), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((c["seqs"], max(n_pages)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(n_pages):
        table[i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    tiles = at * c["kv"] * (c["page"] // 32)
    s = {"case": c, "rows": starts[-1], "n_pages": at, "max_pages": max(n_pages),
         "starts": torch.tensor(starts, dtype=torch.int32, device=DEVICE),
         "lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE), "pages": table.to(DEVICE)}
    shape = (s["rows"], c["heads"], c["dim"])
    kv_shape = (s["rows"], c["kv"], c["dim"])
    rnd = lambda *size: torch.randn(size, generator=g, device=DEVICE)  # noqa: E731
    if c["kind"] == "store":
        s["cache"] = torch.zeros(tiles, _tile_bytes(c), dtype=torch.uint8, device=DEVICE)
        # some channels of keys are much larger than the others, as trained models have them
        s["q"] = rnd(*shape)
        s["k"] = rnd(*kv_shape) * (1 + 4 * (torch.rand(c["kv"], c["dim"], generator=g, device=DEVICE) > 0.95))
        s["v"] = rnd(*kv_shape)
        s["q_out"] = torch.empty_like(s["q"])
    else:
        # codes as a bell-shaped block fills them, scales of keys and values of unit size
        half = 32 * c["dim"] * _bits(c) // 8
        if _bits(c) == 4:
            n = torch.clamp(torch.randn(2, tiles, 2, half, generator=g, device=DEVICE, dtype=torch.float16) * 3 + 8, 0, 15).to(torch.uint8)
            codes = n[0] | n[1] << 4
        else:
            codes = torch.clamp(torch.randn(tiles, 2, half, generator=g, device=DEVICE, dtype=torch.float16) * 48, -127, 127).to(torch.int8)
            codes = codes.view(torch.uint8) ^ 0x80
        unit = 0.33 if _bits(c) == 4 else 0.021
        scales = (unit * (0.6 + 0.8 * torch.rand(tiles, 2, c["dim"], generator=g, device=DEVICE))).half()
        if _bits(c) == 4:
            scales = torch.where(torch.rand(scales.shape, generator=g, device=DEVICE) < 0.5, -scales, scales)
        s["cache"] = torch.cat([torch.cat([codes[:, i], scales[:, i].view(torch.uint8)], 1) for i in (0, 1)], 1)
    if c["kind"] == "attend":
        s["q"] = rnd(*shape) * (1.5 * 8 / math.sqrt(c["dim"]))
        s["out"] = torch.empty_like(s["q"])
        s["sinks"] = rnd(c["heads"]) if c["sinks"] else None
        s["scale"] = 1.0 / math.sqrt(c["dim"])
    else:
        s["k_out"] = torch.empty(kv_shape, device=DEVICE)
        s["v_out"] = torch.empty(kv_shape, device=DEVICE)
    return s


# ---- the plain form

def _positions(s):
    """For each row of the batch: its sequence, its number in it, and its position."""
    row = torch.arange(s["rows"], device=DEVICE)
    seq = torch.searchsorted(s["starts"], row, right=True) - 1
    i = row - s["starts"][seq]
    return seq, i, s["lens"][seq] - (s["starts"][seq + 1] - s["starts"][seq]) + i


def _decode(s):
    """The whole cache as fp32 keys and values, [pages, positions, heads, dim] each.

    A tile is 32 positions of one head.  Keys: 16-byte units of 16 x 4 lanes, a lane's unit
    8 dims of a position for each of two positions (Q4_0) or one (Q8_0) and two blocks;
    scales [16][2][blocks].  Values: 16-byte units of 16 x 4 lanes, a lane's unit 8
    positions of two dims 16 apart, for two blocks (Q4_0) or one (Q8_0); scales
    [blocks][32]."""
    c, b = s["case"], s["cache"]
    n, nb, half = b.shape[0], c["dim"] // 32, 32 * c["dim"] * _bits(c) // 8
    kc, ks, vc, vs = torch.split(b, [half, 64 * nb, half, 64 * nb], 1)
    ks = ks.contiguous().view(torch.float16).float().reshape(n, 4, 4, 2, nb)  # position = 8 * [0] + [1] + 4 * [2]
    ks = ks.permute(0, 1, 3, 2, 4).reshape(n, 32, nb, 1)
    vs = vs.contiguous().view(torch.float16).float().reshape(n, nb, 32).permute(0, 2, 1).unsqueeze(3)
    if _bits(c) == 4:
        k = kc.reshape(n, nb // 2, 4, 4, 4, 2, 2, 2, 2)  # block/2, dims/8, pos/8, pos%4, pos/4%2, block%2, byte/2, byte%2
        k = torch.stack([k & 15, k >> 4], -1).permute(0, 3, 5, 4, 1, 6, 2, 8, 9, 7)
        v = vc.reshape(n, nb // 2, 4, 16, 2, 2, 2, 2)  # block/2, pos/8, dim, block%2, pos/4%2, byte/2, byte%2
        v = torch.stack([v & 15, v >> 4], -1).permute(0, 2, 5, 7, 6, 1, 4, 8, 3)
        k, v = k.to(torch.int8) - 8, v.to(torch.int8) - 8
    else:
        k = (kc ^ 0x80).view(torch.int8).reshape(n, nb // 2, 2, 4, 4, 4, 2, 8)  # block/2, pos/4%2, dims/8, pos/8, pos%4, block%2, dim
        k = k.permute(0, 4, 2, 5, 1, 6, 3, 7)
        v = (vc ^ 0x80).view(torch.int8).reshape(n, nb, 4, 16, 2, 8)  # block, pos/8, dim, dims/16, pos
        v = v.permute(0, 2, 5, 1, 4, 3)
    k = k.reshape(n, 32, nb, 32).float() * ks
    v = v.reshape(n, 32, nb, 32).float() * vs
    paged = lambda x: x.reshape(s["n_pages"], c["kv"], c["page"], c["dim"]).permute(0, 2, 1, 3)  # noqa: E731
    return paged(k), paged(v)


def _angles(c, pos):
    """cos and sin of each position and pair of dims, in 64 bits."""
    h = c["dim"] // 2
    f = ROPE["base"] ** (torch.arange(h, dtype=torch.float64, device=DEVICE) / h)
    edge = [h * math.log(ROPE["original"] / (b * 2 * math.pi)) / math.log(ROPE["base"]) for b in (ROPE["fast"], ROPE["slow"])]
    keep = 1 - torch.clamp((torch.arange(h, dtype=torch.float64, device=DEVICE) - edge[0]) / (edge[1] - edge[0]), 0, 1)
    a = pos.double()[:, None, None] * ((1 - keep) / (ROPE["factor"] * f) + keep / f)
    m = 0.1 * math.log(ROPE["factor"]) + 1
    return a.cos() * m, a.sin() * m


def _rotate(x, cos, sin):
    a, b = x.double().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).float()


def _quantized(c, x):
    """The values that the blocks of 32 of x stand for, in the cache's type: 32-bit steps, in the order that they are defined in."""
    b = x.reshape(-1, 32)
    if _bits(c) == 4:
        top = b.gather(1, b.abs().argmax(1, keepdim=True))
        d = torch.clamp(top / -8, -8188, 8188)
        r = torch.where(d != 0, 1 / d, torch.zeros_like(d))
        q = torch.clamp(torch.floor(b * r + 8.5), 0, 15) - 8
    else:
        d = torch.clamp(b.abs().amax(1, keepdim=True) / 127, max=515.5)
        r = torch.where(d != 0, 1 / d, torch.zeros_like(d))
        t = b * r
        q = torch.clamp(torch.sign(t) * torch.floor(t.abs().double() + 0.5).float(), -127, 127)
    return (q * d.half().float()).reshape(x.shape)


def _store(s):
    cos, sin = _angles(s["case"], _positions(s)[2])
    return {"q": _rotate(s["q"], cos, sin), "k": _quantized(s["case"], _rotate(s["k"], cos, sin)), "v": _quantized(s["case"], s["v"])}


def _read(s):
    seq, _, pos = _positions(s)
    page = s["pages"][seq, pos // s["case"]["page"]].long()
    k, v = _decode(s)
    at = pos % s["case"]["page"]
    return {"k": k[page, at], "v": v[page, at]}


def _attend(s):
    c = s["case"]
    seq, i, pos = _positions(s)
    k, v = _decode(s)
    table = s["pages"].clamp(min=0).long()
    S, T, L, G = c["seqs"], c["new"], s["max_pages"] * c["page"], c["heads"] // c["kv"]
    k, v = (x[table].reshape(S, L, c["kv"], c["dim"]).permute(0, 2, 1, 3).reshape(S * c["kv"], L, c["dim"]) for x in (k, v))
    n = s["starts"][1:] - s["starts"][:-1]
    t = torch.arange(T, device=DEVICE)
    rows = s["starts"][:-1, None] + torch.minimum(t[None], n[:, None] - 1)
    q = s["q"][rows].reshape(S, T, c["kv"], G, c["dim"]).permute(0, 2, 3, 1, 4).reshape(S * c["kv"], G * T, c["dim"])
    scores = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(s["scale"]).reshape(S, c["kv"], G, T, L)
    last = (s["lens"] - n)[:, None] + t[None]  # a row's own position
    j = torch.arange(L, device=DEVICE)
    hidden = j[None, None] > last[:, :, None]
    if c["window"]:
        hidden |= j[None, None] <= last[:, :, None] - c["window"]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    m = scores.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].reshape(1, c["kv"], G, 1, 1)
        m = torch.maximum(m, sink)
    p = scores.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sink - m).exp()
    o = torch.matmul(p.reshape(S * c["kv"], G * T, L), v).reshape(S, c["kv"], G, T, c["dim"]) / total
    return {"out": o.permute(0, 3, 1, 2, 4).reshape(S, T, c["heads"], c["dim"])[seq, i]}


# ---- the framework's operators

_ctx = None


def _plan(s):
    """The handles that a program keeps beside its cache: the context, the descriptors, the workspace."""
    global _ctx
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stream-pt_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import spt
    c = s["case"]
    if _ctx is None:
        _ctx = spt.Context(torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
    cache = spt.KVCache.make(spt.TYPE_Q4_0 if _bits(c) == 4 else spt.TYPE_Q8_0, c["kv"], c["dim"], c["page"], s["n_pages"], s["cache"])
    batch = spt.KVBatch.make(s["starts"], s["lens"], s["pages"], s["rows"], c["new"], c["len"])
    plan = {"cache": cache, "batch": batch}
    if c["kind"] == "store":
        plan["rope"] = spt.Rope(ROPE["base"], ROPE["factor"], ROPE["original"], ROPE["fast"], ROPE["slow"])
    if c["kind"] == "attend":
        n = _ctx.attention_work_bytes(cache, batch, c["heads"], c["window"])
        plan["work"] = torch.empty(n, dtype=torch.uint8, device=DEVICE) if n else None
        plan["sinks"] = None
        if s["sinks"] is not None:
            plan["sinks"] = spt.Tensor.make("attn_sinks", spt.TYPE_F32, [c["heads"]], s["sinks"].data_ptr(), 4 * c["heads"])
    return plan


def run(state):
    s = state
    kind = s["case"]["kind"]
    if not own:
        return {"store": _store, "read": _read, "attend": _attend}[kind](s)
    p = s.get("plan") or s.setdefault("plan", _plan(s))
    if kind == "attend":
        _ctx.attention_batch_into(p["cache"], p["batch"], s["q"], s["out"], s["scale"], window=s["case"]["window"],
                                  sinks=p["sinks"], work=p["work"])
        return {"out": s["out"]}
    if kind == "store":
        _ctx.kv_store_batch(p["cache"], p["batch"], s["k"], s["v"], rope=p["rope"], q=s["q"], q_out=s["q_out"])
    _ctx.kv_load_batch(p["cache"], p["batch"], s["k_out"], s["v_out"])
    out = {"k": s["k_out"], "v": s["v_out"]}
    return {"q": s["q_out"], **out} if kind == "store" else out


# ---- the definition, in 64 bits

def _value(c, tile, pos, dim, values):
    """Keys or values of one tile each, at positions and dims of it (tensors that broadcast): code times scale."""
    nb, half = c["dim"] // 32, 32 * c["dim"] * _bits(c) // 8
    base = half + 64 * nb if values else 0
    blk, e = dim // 32, dim % 32
    scales = base + half
    if values:
        s_at = scales + 2 * (blk * 32 + pos)
        lane = pos // 8 * 16 + e % 16
        if _bits(c) == 4:
            w = pos % 4
            at = (blk // 2 * 64 + lane) * 16 + blk % 2 * 8 + pos // 4 % 2 * 4 + w % 2 * 2 + w // 2
            upper = e // 16
        else:
            at = (blk * 64 + lane) * 16 + e // 16 * 8 + pos % 8
    else:
        row = pos // 8 * 4 + pos % 4
        s_at = scales + 2 * ((row * 2 + pos // 4 % 2) * nb + blk)
        lane = e // 8 * 16 + row
        if _bits(c) == 4:
            w = e % 8
            at = (blk // 2 * 64 + lane) * 16 + pos // 4 % 2 * 8 + blk % 2 * 4 + w % 2 * 2 + w // 4
            upper = w // 2 % 2
        else:
            at = ((blk // 2 * 2 + pos // 4 % 2) * 64 + lane) * 16 + blk % 2 * 8 + e % 8
    byte = lambda x: tile.gather(1, x.reshape(1, -1).expand(tile.shape[0], -1)).long()  # noqa: E731
    code = byte(base + at)
    code = (code >> (4 * upper.reshape(1, -1)) & 15) - 8 if _bits(c) == 4 else code - 128
    bits = byte(s_at) | byte(s_at + 1) << 8
    return code.double() * (bits - (bits >> 15 << 16)).to(torch.int16).view(torch.float16).double()


def _sequence(s, i):
    """Keys and values of all positions of sequence i, [heads, positions, dim], in 64 bits."""
    c = s["case"]
    n = int(s["lens"][i])
    pages = s["pages"][i, :-(-n // c["page"])].long()
    tiles = s["cache"].reshape(s["n_pages"], c["kv"], c["page"] // 32, -1)[pages].permute(1, 0, 2, 3).reshape(-1, _tile_bytes(c))
    pos, dim = torch.arange(32, device=DEVICE)[:, None], torch.arange(c["dim"], device=DEVICE)[None]
    pos, dim = pos + 0 * dim, dim + 0 * pos
    return tuple(_value(c, tiles, pos, dim, values).reshape(c["kv"], -1, c["dim"])[:, :n] for values in (False, True))


def _blocks64(c, x):
    """What the stored blocks of x (fp32) stand for: each step in 64 bits and rounded to the 32 that the format's rule has."""
    f = lambda t: t.float().double()  # noqa: E731
    b = x.double().reshape(-1, 32)
    if _bits(c) == 4:
        big = b.abs().max(1, keepdim=True).values
        first = (b.abs() == big).double() * torch.arange(32, 0, -1, device=DEVICE)
        d = f(torch.take_along_dim(b, first.max(1, keepdim=True).indices, 1) / -8).clamp(-8188, 8188)
        code = (f(f(b * f(1 / d)) + 8.5)).floor().clamp(0, 15) - 8
    else:
        d = f(b.abs().max(1, keepdim=True).values / 127).clamp(max=515.5)
        t = f(b * f(1 / d))
        code = torch.where(t < 0, (t - 0.5).ceil(), (t + 0.5).floor()).clamp(-127, 127)
    return (code.nan_to_num(0) * d.half().double()).reshape(x.shape)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    starts = s["starts"].tolist()
    lens = s["lens"].tolist()
    out = []
    for i, (a, b) in enumerate(zip(starts[:-1], starts[1:])):
        n, first = b - a, lens[i] - (b - a)
        if c["kind"] == "store":
            pairs = torch.arange(c["dim"] // 2, dtype=torch.float64, device=DEVICE)
            plain = torch.exp(-pairs * 2 / c["dim"] * math.log(ROPE["base"]))
            turns = [c["dim"] * math.log(ROPE["original"] / (2 * math.pi * x)) / (2 * math.log(ROPE["base"])) for x in (ROPE["fast"], ROPE["slow"])]
            ramp = ((pairs - turns[0]) / (turns[1] - turns[0])).clamp(0, 1)
            a64 = (first + torch.arange(n, dtype=torch.float64, device=DEVICE))[:, None] * (plain * (1 - ramp) + plain / ROPE["factor"] * ramp)
            turn = torch.polar(torch.full_like(a64, 1 + 0.1 * math.log(ROPE["factor"])), a64)[:, None]
            both = []
            for x in (s["q"][a:b], s["k"][a:b]):
                z = torch.complex(x[..., :c["dim"] // 2].double(), x[..., c["dim"] // 2:].double()) * turn
                both.append(torch.cat([z.real, z.imag], -1))
            out.append({"q": both[0], "k": _blocks64(c, both[1].float()), "v": _blocks64(c, s["v"][a:b])})
            continue
        k, v = _sequence(s, i)
        if c["kind"] == "read":
            out.append({"k": k[:, first:].permute(1, 0, 2), "v": v[:, first:].permute(1, 0, 2)})
            continue
        q = s["q"][a:b].double().reshape(n, c["kv"], -1, c["dim"]).permute(1, 2, 0, 3)
        group = q.shape[1]
        dots = torch.bmm(q.reshape(c["kv"], -1, c["dim"]), k.permute(0, 2, 1).contiguous()).reshape(c["kv"], group, n, -1) * s["scale"]
        behind = (first + torch.arange(n, device=DEVICE))[:, None] - torch.arange(lens[i], device=DEVICE)[None]
        seen = (behind >= 0) & (behind < (c["window"] or lens[i]))
        dots = torch.where(seen, dots, -math.inf)
        if s["sinks"] is not None:
            dots = torch.cat([dots, s["sinks"].double().reshape(c["kv"], group, 1, 1).expand(-1, -1, n, 1)], -1)
        p = torch.softmax(dots, -1)[..., :lens[i]]
        o = torch.bmm(p.reshape(c["kv"], group * n, -1), v.contiguous()).reshape(c["kv"], group, n, -1)
        out.append({"out": o.permute(2, 0, 1, 3).reshape(n, c["heads"], c["dim"])})
    return {name: torch.cat([o[name] for o in out]) for name in out[0]}
