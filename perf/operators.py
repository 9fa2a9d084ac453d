"""Timed cases of the 4-bit paged KV cache: appending rows (rotation on the way) and attention over the pages.

``run`` computes an operator in plain torch operations, or through the
package's entry points when ``own`` is true.  Both sides work on the same
pool of pages in the cache's byte layout:

  pool [page][kv head][block], a block holding ``P`` tokens of one head:
    K codes    P rows of D/2 bytes, channel 2b in the low half of byte b
    K scales   per token and group of 32 channels two f16: s, o
    V codes    as K, but rows of 2 (D = 128) or 4 (D = 64) tokens share a
               128-byte line and the 32-byte quarters of a line are permuted
    V scales   per pair of tokens and group: s, o, s', o'
  value = s * (1 + code / 16) + o

For a group of 32 channels with least and largest value lo, hi (each clamped
to +-20000): s = f16((hi - lo) * 16/15), o = f16(lo - s) and
code = clamp(round((x - o) * (16 / s) - 16), 0, 15).
"""

import importlib
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LIMIT = 20000.0
DEV = "cuda"


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _case(name, kind, heads, kv_heads, dim, page, dtype, seqs, kv, rows, tree=False, half=True, shape=1):
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "seqs": seqs,
         "kv_min": kv[0], "kv_max": kv[1], "rows_min": rows[0], "rows_max": rows[1], "tree": tree, "half": half,
         "shape": shape}
    return {"name": name, **c} if name else c


def listed():
    return [
        # One decoded token of one sequence (Llama-3-8B heads): the append of the
        # batch-1 loop, all launch latency.
        _case("append_1", "append", 32, 8, 128, 64, "bf16", 1, (2048, 2048), (1, 1), half=False),
        # A serving step of 64 decoding sequences with Qwen2.5-7B heads, 16-token pages.
        _case("append_64x1", "append", 28, 4, 128, 16, "f16", 64, (100, 12000), (1, 1)),
        # k + 1 = 5 verify rows each of 37 sequences, f32 rows as the quantized
        # matmul returns them, Llama-3.2-1B heads.
        _case("append_37x5_f32", "append", 32, 8, 64, 32, "f32", 37, (17, 4000), (5, 5), half=False),
        # The rows of a long prompt.
        _case("append_8192", "append", 32, 8, 128, 64, "bf16", 1, (0, 0), (8192, 8192)),
        # One token against a short context: attention's launch latency.
        _case("decode_1x2048", "attend", 32, 8, 128, 64, "bf16", 1, (2047, 2047), (1, 1)),
        # The framework's headline step: 5 verify rows against 2048 tokens.
        _case("verify_1x5_2048", "attend", 32, 8, 128, 64, "bf16", 1, (2048, 2048), (5, 5)),
        # One sequence at a long context.
        _case("decode_1x131072", "attend", 32, 8, 128, 128, "bf16", 1, (131071, 131071), (1, 1)),
        # A full serving batch, lengths mixed.
        _case("decode_64_mixed", "attend", 32, 8, 128, 64, "bf16", 64, (500, 16000), (1, 1)),
        # k = 8 speculation for 24 sequences, Qwen2.5-7B heads (7 query heads share a KV head).
        _case("verify_24x9_mixed", "attend", 28, 4, 128, 16, "f16", 24, (300, 9000), (9, 9)),
        # The 60-node draft tree against 4096 tokens.
        _case("tree_60_4096", "attend", 32, 8, 128, 64, "bf16", 1, (4096, 4096), (60, 60), tree=True),
        # A prompt's 2048-row chunk after 6144 cached tokens.
        _case("chunk_2048_6144", "attend", 32, 8, 128, 64, "bf16", 1, (6144, 6144), (2048, 2048)),
        # The whole step of a small model (Qwen2.5-0.5B heads, head size 64): 8
        # sequences verify draft trees of 1 to 31 nodes, append then attention.
        _case("step_8_trees_64", "step", 14, 2, 64, 32, "bf16", 8, (0, 1500), (1, 31), tree=True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    heads, kv_heads, dim = rng.choice([(32, 8, 128), (28, 4, 128), (14, 2, 64), (32, 8, 64), (8, 8, 128), (16, 1, 128)])
    kind = rng.choice(["append", "attend", "attend", "attend", "step"])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "f16"] if kind == "attend" else ["bf16", "f16", "f32"])
    half = rng.random() < 0.7
    shape = rng.randrange(1, 1 << 20)
    form = rng.choice(["decode", "verify", "tree", "chunk"])
    if form == "decode":
        seqs, r0, r1 = log_int(1, 64), 1, 1
    elif form == "verify":
        seqs, r0 = log_int(1, 32), rng.randrange(1, 4)
        r1 = r0 + rng.randrange(0, 13)
    elif form == "tree":
        seqs, r0, r1 = log_int(1, 8), rng.randrange(1, 20), rng.randrange(20, 65)
    else:
        seqs, r0 = 1, log_int(65, 2000)
        r1 = r0
    # At most 400000 cached tokens, and the row-key products of a 2048-row chunk over 7168 keys.
    most = min(100000, 400000 // seqs, 2048 * 7168 * 32 * 128 // (seqs * r1 * heads * dim))
    kv_max = log_int(33, max(64, most if form != "chunk" else min(most, 6000)))
    kv_min = max(0, min(kv_max, log_int(1, kv_max) - 1))
    return _case(None, kind, heads, kv_heads, dim, page, dtype, seqs, (kv_min, kv_max), (r0, r1), form == "tree", half,
                 shape)


def _shape(c):
    """Lengths, rows, positions and ancestor masks of a case (the same for every seed)."""
    r = random.Random(c["shape"] * 7919 + 13)
    kv = [r.randint(c["kv_min"], c["kv_max"]) for _ in range(c["seqs"])]
    rows = [r.randint(c["rows_min"], c["rows_max"]) for _ in range(c["seqs"])]
    pos, masks = [], []
    for n, m in zip(kv, rows):
        depth, anc = [], []
        for i in range(m):
            if not c["tree"]:
                depth.append(i)
            elif i == 0:
                depth.append(0)
                anc.append(1)
            else:
                p = r.randrange(max(0, i - 10), i)  # BFS order, at most 10 candidates a node
                depth.append(depth[p] + 1)
                anc.append(anc[p] | (1 << i))
        pos += [n + d for d in depth]
        masks += anc
    return kv, rows, pos, masks if c["tree"] else None


def work(c):
    kv, rows, _, masks = _shape(c)
    hq, hk, d = c["heads"], c["kv_heads"], c["dim"]
    size = 4 if c["dtype"] == "f32" else 2
    total = sum(rows)
    token = hk * d * 10 // 8  # bytes of a token's K and V of all heads: 5 bits an element
    b = f = 0
    if c["kind"] != "attend":
        # q in and out, k and v in, 4-bit rows and the values they stand for out, the rotation's table rows
        b += total * (hq * d * (size + 2) + 2 * hk * d * size + token + 2 * hk * d * 2 + d * 4)
        f += total * ((hq + hk) * d * 3 + 2 * hk * d * 8)
    if c["kind"] != "append":
        b += sum(n + m for n, m in zip(kv, rows)) * token + 2 * total * hq * d * 2
        pairs, at = 0, 0
        for n, m in zip(kv, rows):
            pairs += n * m + (sum(bin(x).count("1") for x in masks[at:at + m]) if masks else m * (m + 1) // 2)
            at += m
        f += 4 * d * hq * pairs
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------------------
# The byte layout
# ---------------------------------------------------------------------------
def _maps(p, d):
    """Byte offsets inside a block: K codes [p, d/2], K scales [p, g, 4], V codes, V scales; and the block's size."""
    j = torch.arange(p, device=DEV)[:, None]
    b = torch.arange(d // 2, device=DEV)[None]
    if d == 128:
        v = (j // 2) * 128 + 32 * (((j % 2) * 2 + b // 32) ^ ((j // 2) % 4)) + b % 32
    else:
        v = (j // 4) * 128 + 32 * ((j % 4) ^ ((j // 4) % 2)) + b
    g = torch.arange(d // 32, device=DEV)[None, :, None]
    e = torch.arange(4, device=DEV)[None, None]
    jj, n = j[..., None], d // 32
    codes, scales = p * d // 2, p * n * 4
    ks = codes + jj * n * 4 + g * 4 + e
    vs = 2 * codes + scales + (jj // 2) * n * 8 + g * 8 + (jj % 2) * 4 + e
    return j * (d // 2) + b, ks, codes + scales + v, vs, 2 * (codes + scales)


def _quantize(x):
    """x [..., d] f32 -> codes [..., d] uint8, (s, o) [..., d/32, 2] f16."""
    g = x.clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) * (16.0 / 15.0)).half()
    o = (lo - s.float()).half()
    inv = torch.where(s > 0, 16.0 / s.float(), torch.zeros_like(lo))
    c = torch.round((g - o.float()) * inv - 16.0).clamp(0, 15).nan_to_num(0.0)
    return c.to(torch.uint8).flatten(-2), torch.cat([s, o], -1)


def _dequantize(codes, so):
    so = so.float()
    v = so[..., :1] * (1.0 + codes.unflatten(-1, (-1, 32)).float() / 16.0) + so[..., 1:]
    return v.flatten(-2)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _bytes(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _halves(b):
    """uint8 [..., 4] -> f16 [..., 2]."""
    return b.contiguous().view(torch.float16)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _rows_like(gen, n, h, d, spread):
    """Rows as a model's projections give them: normal, with a few strong channels per head."""
    x = torch.randn(n, h, d, device=DEV, generator=gen)
    strong = (torch.rand(1, h, d, device=DEV, generator=gen) < 0.04).float()
    return x * 0.9 + strong * spread * torch.randn(1, h, d, device=DEV, generator=gen)


def prepare(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    host = random.Random(seed)
    hq, hk, d, p = c["heads"], c["kv_heads"], c["dim"], c["page"]
    kv, rows, pos, masks = _shape(c)
    total = sum(rows)
    need = [(n + m + p - 1) // p for n, m in zip(kv, rows)]
    n_pages = sum(need) + 3
    order = list(range(n_pages))
    host.shuffle(order)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (max(need) - n))
        at += n
    st = {"case": c, "hq": hq, "hk": hk, "d": d, "p": p, "n_pages": n_pages, "half": c["half"],
          "maps": _maps(p, d), "scale": 1.0 / math.sqrt(d)}
    block = st["maps"][4]
    # The pool: every slot that holds a token gets quantized rows, the others bytes that read as NaN.
    pool = torch.full((n_pages, hk, block), 255, dtype=torch.uint8, device=DEV)
    filled = [n + (m if c["kind"] == "attend" else 0) for n, m in zip(kv, rows)]
    slots_of = torch.zeros(n_pages, dtype=torch.long)
    for t, n, f in zip(table, need, filled):
        for i in range(n):
            slots_of[t[i]] = max(0, min(p, f - i * p))
    used = slots_of.to(DEV)
    kc, ks, vc, vs, _ = st["maps"]
    step = max(1, (1 << 26) // (hk * p * d))
    for a in range(0, n_pages, step):
        m = min(step, n_pages - a)
        part = torch.full((m, hk, block), 255, dtype=torch.uint8, device=DEV)
        live = torch.arange(p, device=DEV)[None] < used[a:a + m, None]
        live = live[:, None, :, None]
        for cm, sm, spread in ((kc, ks, 5.0), (vc, vs, 1.0)):
            x = _rows_like(gen, m * p, hk, d, spread).view(m, p, hk, d).transpose(1, 2)
            codes, so = _quantize(x)
            by = torch.where(live, _bytes(codes), torch.full_like(_bytes(codes), 255))
            part[:, :, cm.flatten()] = by.flatten(2)
            sb = so.contiguous().view(torch.uint8)
            sb = torch.where(live[..., None], sb, torch.full_like(sb, 255))
            part[:, :, sm.flatten()] = sb.flatten(2)
        pool[a:a + m] = part
    st["pool"] = pool
    # The new rows: views of one fused projection output for the append.
    dt = DTYPES[c["dtype"]]
    st["out_dtype"] = torch.bfloat16 if dt == torch.float32 else dt
    fused = torch.cat([_rows_like(gen, total, hq, d, 1.5) * 1.3, _rows_like(gen, total, hk, d, 5.0),
                       _rows_like(gen, total, hk, d, 1.0)], 1).to(dt)
    st["q"], st["k"], st["v"] = fused[:, :hq], fused[:, hq:hq + hk], fused[:, hq + hk:]
    if c["kind"] == "attend":
        st["q"] = st["q"].contiguous()
    # Rotation tables.
    n_pos = max(n + m for n, m in zip(kv, rows)) + 1
    freq = 1.0 / (500000.0 ** (torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d))
    angle = torch.arange(n_pos, device=DEV, dtype=torch.float64)[:, None] * freq
    st["cos"], st["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    # Index arrays of the plain form; the package's plan is made from the same lists.
    seq = [b for b, m in enumerate(rows) for _ in range(m)]
    idx = [i for m in rows for i in range(m)]
    dev = lambda v: torch.tensor(v, dtype=torch.long, device=DEV)  # noqa: E731
    st["seq"], st["idx"], st["pos"], st["table"] = dev(seq), dev(idx), dev(pos), dev(table)
    st["kv"], st["rows"], st["max_rows"] = dev(kv), dev(rows), max(rows)
    st["slot"] = st["kv"][st["seq"]] + st["idx"]
    signed = [m - (1 << 64) if m >> 63 else m for m in masks] if masks else None
    st["masks"] = dev(signed) if masks else None
    st["q_out"] = torch.empty(total, hq, d, dtype=st["out_dtype"], device=DEV)
    st["k_out"] = torch.empty(total, hk, d, dtype=torch.float16, device=DEV)
    st["v_out"] = torch.empty_like(st["k_out"])
    st["out"] = torch.empty(total, hq, d, dtype=st["out_dtype"], device=DEV)
    if own:
        pkg = importlib.import_module("abyo-speculate_b200")
        cache = pkg.KV4Cache(pool, n_layers=1, n_heads=hq, n_kv_heads=hk, head_dim=d, page_tokens=p, n_pages=n_pages,
                             rope=(st["cos"], st["sin"]), rope_half=c["half"])
        st["batch"] = pkg.KV4Batch(cache)
        st["batch"].plan(kv, rows, table, positions=pos, masks=masks)
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _rotate(x, cos, sin, half):
    c, s = cos[:, None], sin[:, None]
    if half:
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)


def _plain_append(st):
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    q = _rotate(st["q"].float(), cos, sin, st["half"])
    k = _rotate(st["k"].float(), cos, sin, st["half"])
    kc, ks, vc, vs, block = st["maps"]
    p, hk = st["p"], st["hk"]
    page = st["table"][st["seq"], st["slot"] // p]
    j = st["slot"] % p
    base = (page[:, None] * hk + torch.arange(hk, device=DEV)) * block
    flat = st["pool"].view(-1)
    out = []
    for x, cm, sm in ((k, kc, ks), (st["v"].float(), vc, vs)):
        codes, so = _quantize(x)
        flat[base[..., None] + cm[j][:, None]] = _bytes(codes)
        flat[base[..., None, None] + sm[j][:, None]] = so.contiguous().view(torch.uint8)
        out.append(_dequantize(codes, so).half())
    return q.to(st["out_dtype"]), out[0], out[1]


def _plain_attend(st, q):
    hq, hk, d, p = st["hq"], st["hk"], st["d"], st["p"]
    kc, ks, vc, vs, _ = st["maps"]
    n, width = st["table"].shape
    t = width * p
    blocks = st["pool"][st["table"]].transpose(1, 2)  # [seqs, kv heads, pages, block]
    live = (torch.arange(t, device=DEV)[None] < (st["kv"] + st["rows"])[:, None])[:, None, :, None]

    def values(cm, sm):
        codes = _nibbles(blocks[..., cm])
        x = _dequantize(codes, _halves(blocks[..., sm]).view(*codes.shape[:-1], d // 32, 2)).flatten(2, 3)
        return torch.where(live, x, torch.zeros((), device=DEV))

    g, m = hq // hk, st["max_rows"]
    qp = torch.zeros(n, m, hq, d, device=DEV)
    qp[st["seq"], st["idx"]] = q.float()
    qp = qp.view(n, m, hk, g, d).permute(0, 2, 3, 1, 4).reshape(n, hk, g * m, d)
    s = (qp @ values(kc, ks).transpose(-1, -2)) * st["scale"]
    at = torch.arange(t, device=DEV)[None, None]
    j = at - st["kv"][:, None, None]
    i = torch.arange(m, device=DEV)[None, :, None]
    if st["masks"] is None:
        see = j <= i
    else:
        bits = torch.zeros(n, m, dtype=torch.long, device=DEV)
        bits[st["seq"], st["idx"]] = st["masks"]
        see = (j < 0) | ((j < 64) & (((bits[..., None] >> j.clamp(0, 63)) & 1) == 1))
    see = see & (at < (st["kv"] + st["rows"])[:, None, None])
    s = s.view(n, hk, g, m, t).masked_fill(~see[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    o = (e.view(n, hk, g * m, t) @ values(vc, vs)).view(n, hk, g, m, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(n, m, hq, d)
    return o[st["seq"], st["idx"]].to(st["out_dtype"])


def run(st):
    kind = st["case"]["kind"]
    out, q = [], st["q"]
    if own:
        if kind != "attend":
            st["batch"].append(0, q, st["k"], st["v"], q_out=st["q_out"], k_out=st["k_out"], v_out=st["v_out"])
            out, q = [st["q_out"], st["k_out"], st["v_out"]], st["q_out"]
        if kind != "append":
            out.append(st["batch"].attend(0, q, out=st["out"]))
        return out
    if kind != "attend":
        out = list(_plain_append(st))
        q = out[0]
    if kind != "append":
        out.append(_plain_attend(st, q))
    return out


# ---------------------------------------------------------------------------
# The definition in 64 bits, element by element
# ---------------------------------------------------------------------------
def _address(d, p, j, ch, value):
    """Byte offset and nibble of element (token j, channel ch) in a block, and of its group's s."""
    by, g = ch // 2, ch // 32
    area = p * d // 2 + p * d // 8
    if not value:
        return j * (d // 2) + by, p * d // 2 + (j * (d // 32) + g) * 4
    line = 256 // d  # tokens of a 128-byte line
    quarter = (j % line) * (d // 64) + by // 32
    turn = (j // line) % (4 if d == 128 else 2)
    return (area + (j // line) * 128 + (quarter ^ turn) * 32 + by % 32,
            area + p * d // 2 + (j // 2) * (d // 32) * 8 + g * 8 + (j % 2) * 4)


def _half_bits(lo, hi):
    bits = lo.long() | (hi.long() << 8)
    e, m = (bits >> 10) & 31, (bits & 1023).double()
    sign = torch.where(bits >> 15 == 1, -1.0, 1.0).double()
    return sign * torch.where(e == 0, m * 2.0 ** -24, (1024 + m) * torch.exp2((e - 25).double()))


def _read_64(st, b, n, value):
    """Values [n tokens, kv heads, d] of sequence b in 64 bits."""
    d, p, hk, block = st["d"], st["p"], st["hk"], st["maps"][4]
    t = torch.arange(n, device=DEV)
    ch = torch.arange(d, device=DEV)
    at, sc = _address(d, p, (t % p)[:, None, None], ch[None, None], value)
    base = ((st["table"][b, t // p] * hk)[:, None] + torch.arange(hk, device=DEV))[..., None] * block
    flat = st["pool"].view(-1)
    code = (flat[base + at] >> (4 * (ch % 2)).to(torch.uint8)) & 15
    s = _half_bits(flat[base + sc], flat[base + sc + 1])
    o = _half_bits(flat[base + sc + 2], flat[base + sc + 3])
    return s * (16 + code.double()) / 16 + o


def _exact_attend(st, q, new=None):
    hq, hk, d = st["hq"], st["hk"], st["d"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    kv, rows = st["kv"].tolist(), st["rows"].tolist()
    at = 0
    for b, (n, m) in enumerate(zip(kv, rows)):
        k, v = (_read_64(st, b, n + (0 if new else m), x) for x in (False, True))
        if new:
            k, v = torch.cat([k, new[0][at:at + m]]), torch.cat([v, new[1][at:at + m]])
        see = torch.ones(m, n + m, dtype=torch.bool, device=DEV)
        tail = torch.ones(m, m, dtype=torch.bool, device=DEV).tril()
        if st["masks"] is not None:
            bits = st["masks"][at:at + m]
            tail = torch.stack([(bits >> i) & 1 for i in range(m)], 1) == 1
        see[:, n:] = tail
        for h in range(hq):
            s = q[at:at + m, h].double() @ k[:, h * hk // hq].T * st["scale"]
            out[at:at + m, h] = torch.softmax(s.masked_fill(~see, -math.inf), -1) @ v[:, h * hk // hq]
        at += m
    return out


def _exact_append(st):
    d = st["d"]
    c, s = st["cos"].double()[st["pos"]], st["sin"].double()[st["pos"]]
    first = torch.arange(d // 2, device=DEV) if st["half"] else torch.arange(0, d, 2, device=DEV)
    second = first + (d // 2 if st["half"] else 1)

    def turn(x):
        y, x = torch.empty(x.shape, dtype=torch.float64, device=DEV), x.double()
        y[..., first] = x[..., first] * c[:, None] - x[..., second] * s[:, None]
        y[..., second] = x[..., second] * c[:, None] + x[..., first] * s[:, None]
        return y

    def stored(x):
        x = x.clamp(-LIMIT, LIMIT).reshape(*x.shape[:-1], d // 32, 32)
        lo = x.min(-1, keepdim=True).values
        a = ((x.max(-1, keepdim=True).values - lo) * 16 / 15).half().double()
        o = (lo - a).half().double()
        code = torch.where(a > 0, (16 * (x - o) / torch.where(a > 0, a, 1.0) - 16).round().clamp(0, 15), 0.0)
        return (a * (16 + code) / 16 + o).reshape(*x.shape[:-2], d)

    return turn(st["q"]), stored(turn(st["k"])), stored(st["v"].double())


def exact(c, seed):
    st = prepare(c, seed)
    kind = c["kind"]
    out, q, new = [], st["q"], None
    if kind != "attend":
        out = list(_exact_append(st))
        # The attention of a step reads the rotated queries as they were rounded and the values as they were stored.
        q, new = out[0].to(st["out_dtype"]), (out[1], out[2])
    if kind != "append":
        out.append(_exact_attend(st, q, new))
    return out
