"""Cases of the 4-bit KV cache: quantising rows as they are written, reading them back, rolling the context, and the
decode and prefill attention that read it.  `run` makes either the plain torch form of an operator (`own` false) or the
calls of the library (`own` true).

The format.  A cache holds one layer as uint8 [n_kv][ceil(n_ctx / 16)][block bytes]; a block is 16 consecutive positions
of one kv head.  Every head row is cut into groups of 64 dims; a group keeps two fp16 numbers, an offset m and a step d,
and one 4-bit code per value, which stands for m + d * code:

    m = fp16(min x)     d = fp16(max(0, (max x - m) / 15))     code = clamp(round((x - m) / d), 0, 15)   (0 where d = 0)

evaluated exactly and rounded once where it says fp16 (to nearest, ties to even, as round does).  Bytes of a block, with
hd = head_dim, NG = hd / 64:

    [0, 8 hd)           K codes: row s at 32-bit word s * hd/8; word t * hd/32 + i of a row (t < 4) holds dims
                        32 i + 8 t + e, e = 0..7, dim e in bits 4e..4e+3
    [8 hd, 16 hd)       V codes: one byte per (row, pair of dims 2p, 2p+1), the even dim in the low half; with
                        p = 8 j + r and row s = 8 h + 2 t + u the byte is at (j/4) * 512 + (4 r + t) * 16 + (j%4) * 4 + 2 u + h
    [16 hd, 16 hd + 64 NG)      K scales: fp16 [16 rows][NG][d, m];    then the V scales, the same
"""
import math

import numpy as np
import torch

own = False

ROPE_NORMAL, ROPE_NEOX = 0, 1


# ---------------------------------------------------------------------------------------------------------- cases
def _decode(name, n_head, n_kv, head_dim, length, append, rope_type=ROPE_NEOX, theta=1e6):
    c = {"op": "decode", "n_head": n_head, "n_kv": n_kv, "head_dim": head_dim, "length": length, "append": append,
         "rope_type": rope_type, "theta": theta}
    return dict(c, name=name) if name else c


def _prefill(name, n_head, n_kv, head_dim, n_past, batch, rope_type=ROPE_NORMAL, theta=5e5):
    c = {"op": "prefill", "n_head": n_head, "n_kv": n_kv, "head_dim": head_dim, "n_past": n_past, "batch": batch,
         "rope_type": rope_type, "theta": theta}
    return dict(c, name=name) if name else c


def _store(name, n_kv, head_dim, pos, batch):
    c = {"op": "store", "n_kv": n_kv, "head_dim": head_dim, "pos": pos, "batch": batch}
    return dict(c, name=name) if name else c


def _load(name, n_kv, head_dim, n_ctx, row, rows):
    c = {"op": "load", "n_kv": n_kv, "head_dim": head_dim, "n_ctx": n_ctx, "row": row, "rows": rows}
    return dict(c, name=name) if name else c


def _roll(name, n_layer, n_kv, head_dim, n_ctx, n_keep, shift):
    c = {"op": "roll", "n_layer": n_layer, "n_kv": n_kv, "head_dim": head_dim, "n_ctx": n_ctx, "n_keep": n_keep, "shift": shift}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the first token of a conversation: one position, one row appended; nothing but latency
        _decode("decode_first_token", 12, 2, 128, 1, True),
        # a decode step early in a conversation, the new row appended in the same call
        _decode("decode_1k_append", 28, 4, 128, 1024, True),
        # 64-dim heads, a ragged length, over a cache that is already complete (only q is rotated)
        _decode("decode_32k_hd64", 32, 8, 64, 32001, False),
        # long-context decode: the streaming case, 302 MB of cache
        _decode("decode_1m", 16, 2, 128, 1048576, False),
        # a short prompt at the start of an empty cache
        _prefill("prefill_prompt", 12, 2, 128, 0, 45, ROPE_NEOX, 1e6),
        # a full chunk behind 8192 rows
        _prefill("prefill_512_at_8k", 32, 8, 128, 8192, 512),
        # a chunk written by the unfused call at an odd position, and the rows it left read back
        _store("store_chunk", 8, 128, 1001, 512),
        # a whole long prompt taken over into the cache, and read back
        _store("store_8k", 8, 128, 0, 8192),
        # a few hundred rows of 64-dim heads, from inside a block to inside a block
        _load("load_ragged", 4, 64, 2000, 5, 777),
        # a long prefix turned back into an fp16 cache
        _load("load_32k", 8, 128, 32768, 0, 32768),
        # a conversation forked from a shared cache and rolled by an odd number of rows: one small layer
        _roll("roll_small", 1, 2, 128, 1000, 4, 333),
        # the same for the layers of a model, half of the context dropped
        _roll("roll_layers", 8, 8, 128, 8192, 5, 4094),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    hd = rng.choice([64, 128, 128])
    n_kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    op = rng.choice(["decode", "decode", "prefill", "store", "load", "roll"])
    rope = (rng.choice([ROPE_NORMAL, ROPE_NEOX]), rng.choice([1e4, 5e5, 1e6]))
    if op == "decode":
        return _decode(None, n_kv * group, n_kv, hd, log_int(1, 1048576 // n_kv), rng.random() < 0.5, *rope)
    if op == "prefill":
        batch = log_int(1, 512)
        return _prefill(None, n_kv * min(group, 8 if n_kv < 8 else 4), n_kv, hd, rng.choice([0, log_int(1, 8192)]), batch, *rope)
    if op == "store":
        return _store(None, n_kv, hd, rng.randrange(0, 4096), log_int(1, 8192))
    if op == "load":
        n_ctx = log_int(16, 32768)
        row = rng.randrange(0, n_ctx)
        return _load(None, n_kv, hd, n_ctx, row, rng.randint(1, n_ctx - row))
    n_ctx = log_int(16, 8192)
    n_keep = rng.randrange(0, n_ctx // 2)
    return _roll(None, rng.randint(1, 8), n_kv, hd, n_ctx, n_keep, rng.randint(1, n_ctx - n_keep))


def _row_bytes(hd):
    return hd // 2 + hd // 16         # codes and scales of one row of K or of V


def work(c):
    op, hd, n_kv = c["op"], c["head_dim"], c["n_kv"]
    row4 = 2 * n_kv * _row_bytes(hd)              # one position of the 4-bit cache
    row16 = 2 * n_kv * hd * 2                     # the same as fp16
    row32 = 2 * n_kv * hd * 4                     # as fp32 activations
    if op == "decode":
        n = c["length"] * row4 + 2 * c["n_head"] * hd * 4
        if c["append"]:
            n += row32 + row16                    # the new row comes in, and its values go out again
        return {"bytes": n, "flops": 4 * c["n_head"] * hd * c["length"]}
    if op == "prefill":
        b, past = c["batch"], c["n_past"]
        pairs = b * past + b * (b + 1) // 2
        return {"bytes": (past + b) * row4 + b * (c["n_head"] * hd * (4 + 2) + row32 + row16), "flops": 4 * c["n_head"] * hd * pairs}
    if op == "store":
        return {"bytes": c["batch"] * (row32 + row4 + row16), "flops": 0}
    if op == "load":
        return {"bytes": c["rows"] * (row4 + row16), "flops": 0}
    return {"bytes": c["n_layer"] * c["n_ctx"] * (2 * row4 + row16), "flops": 0}


# ---------------------------------------------------------------------------------------------------------- inputs
def _blocks(n_ctx):
    return (n_ctx + 15) // 16


def _channels(gen, heads, hd):
    """Spread and offset of the channels of a key or value head: most alike, a few with a large offset."""
    spread = torch.exp(0.4 * torch.randn(heads, 1, hd, device="cuda", generator=gen))
    offset = 4.0 * torch.randn(heads, 1, hd, device="cuda", generator=gen) * (torch.rand(heads, 1, hd, device="cuda", generator=gen) < 0.05)
    return spread, offset


def _cache(gen, heads, hd, n_ctx, rows):
    """A cache whose first `rows` rows hold quantised values; the rest is whatever the memory held."""
    n_blk, ng = _blocks(n_ctx), hd // 64
    used = _blocks(rows)
    cache = torch.randint(0, 256, (heads, n_blk, 2 * 16 * _row_bytes(hd)), dtype=torch.uint8, device="cuda", generator=gen)
    if rows == 0:
        return cache
    parts = []
    for _ in range(2):
        spread, offset = _channels(gen, heads, hd)
        x = torch.randn(heads, used * 16, hd, device="cuda", generator=gen) * spread + offset
        g = x.view(heads, used * 16, ng, 64)
        m = g.amin(-1, keepdim=True).half().float()
        d = ((g.amax(-1, keepdim=True) - m) / 15).half().float()
        code = ((g - m) / d).round_().clamp_(0, 15).to(torch.uint8).view(heads, used, 16, hd)
        parts.append((code, torch.cat((d, m), -1).half().view(heads, used, 16 * ng * 2).view(torch.uint8)))
    (kcode, kscale), (vcode, vscale) = parts
    # [row][i][t][byte][half] -> [row][t][i][byte]
    k = kcode.view(heads, used, 16, hd // 32, 4, 4, 2)
    k = (k[..., 0] | (k[..., 1] << 4)).transpose(3, 4).reshape(heads, used, 8 * hd)
    # [h][t][u] rows, [j/4][j%4][r][half] dims -> [j/4][r][t][j%4][u][h]
    v = vcode.view(heads, used, 2, 4, 2, hd // 64, 4, 8, 2)
    v = (v[..., 0] | (v[..., 1] << 4)).permute(0, 1, 5, 7, 3, 6, 4, 2).reshape(heads, used, 8 * hd)
    image = torch.cat((k, v, kscale, vscale), -1)
    fill = (rows % 16) or 16                      # rows of the last block that are written
    if fill == 16:
        cache[:, :used] = image
    else:
        cache[:, : used - 1] = image[:, :-1]
        # rows behind the last one keep what the memory held: NaN scales among it
        last, s0 = image[:, -1].clone(), 16 * hd
        rest = torch.full((heads, 2, 16, 4 * ng), 255, dtype=torch.uint8, device="cuda")
        scales = last[:, s0:].view(heads, 2, 16, 4 * ng)
        scales[:, :, fill:] = rest[:, :, fill:]
        cache[:, used - 1] = last
    return cache


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, hd, n_kv = c["op"], c["head_dim"], c["n_kv"]
    s = {"case": c}

    def rows(n):
        spread, offset = _channels(gen, n_kv, hd)
        return torch.randn(n, n_kv, hd, device="cuda", generator=gen) * spread.view(1, n_kv, hd) + offset.view(1, n_kv, hd)

    def halves(heads, n):
        return [torch.zeros(heads, n, hd, dtype=torch.float16, device="cuda") for _ in range(2)]

    if op == "decode":
        s["n_ctx"] = 16 * _blocks(c["length"]) + 16
        s["cache"] = _cache(gen, n_kv, hd, s["n_ctx"], c["length"] - 1 if c["append"] else c["length"])
        s["q"] = torch.randn(c["n_head"], hd, device="cuda", generator=gen)
        s["k"], s["v"] = rows(1)[0], rows(1)[0]
        s["pos"] = torch.tensor([c["length"] - 1], dtype=torch.int32, device="cuda")
        s["out"] = torch.zeros(c["n_head"], hd, device="cuda")
        s["kh"], s["vh"] = halves(n_kv, 1)
    elif op == "prefill":
        s["n_ctx"] = c["n_past"] + c["batch"] + 7
        s["cache"] = _cache(gen, n_kv, hd, s["n_ctx"], c["n_past"])
        s["q"] = torch.randn(c["batch"], c["n_head"], hd, device="cuda", generator=gen)
        s["k"], s["v"] = rows(c["batch"]), rows(c["batch"])
        s["out"] = torch.zeros(c["batch"], c["n_head"], hd, dtype=torch.float16, device="cuda")
        s["kh"], s["vh"] = halves(n_kv, c["batch"])
    elif op == "store":
        s["n_ctx"] = c["pos"] + c["batch"] + 3
        s["cache"] = _cache(gen, n_kv, hd, s["n_ctx"], c["pos"])
        s["k"], s["v"] = rows(c["batch"]), rows(c["batch"])
        s["kh"], s["vh"] = halves(n_kv, c["batch"])
    elif op == "load":
        s["n_ctx"] = c["n_ctx"]
        s["cache"] = _cache(gen, n_kv, hd, c["n_ctx"], c["n_ctx"])
        s["kh"], s["vh"] = halves(n_kv, c["rows"])
    else:
        heads = c["n_layer"] * n_kv
        s["n_ctx"] = c["n_ctx"]
        s["shared"] = _cache(gen, heads, hd, c["n_ctx"], c["n_ctx"])
        s["cache"] = torch.zeros_like(s["shared"])
        s["kh"], s["vh"] = halves(heads, c["n_ctx"])
    return s


# ---------------------------------------------------------------------------------------------------------- plain form
def _values(cache, hd):
    """The fp32 values of every row of a cache: K, V [heads][16 * blocks][hd]."""
    heads, n_blk = cache.shape[:2]
    ng = hd // 64

    def scaled(code, at):
        scale = cache[:, :, at: at + 64 * ng].contiguous().view(torch.float16).view(heads, n_blk, 16, ng, 2).float()
        code = code.reshape(heads, n_blk, 16, ng, 64).float()
        return (scale[..., 1:] + scale[..., :1] * code).view(heads, n_blk * 16, hd)

    k = cache[:, :, : 8 * hd].reshape(heads, n_blk, 16, 4, hd // 32, 4)
    k = torch.stack((k & 15, k >> 4), -1).transpose(3, 4)
    v = cache[:, :, 8 * hd: 16 * hd].reshape(heads, n_blk, hd // 64, 8, 4, 4, 2, 2)
    v = torch.stack((v & 15, v >> 4), -1).permute(0, 1, 7, 4, 6, 2, 5, 3, 8)
    return scaled(k, 16 * hd), scaled(v, 16 * hd + 64 * ng)


def _to_half(x):
    """float64 -> the nearest fp16 number, in one rounding, as float64."""
    power = (x.contiguous().view(torch.int64) & (0x7FF << 52)).view(torch.float64)      # 2^floor(log2 |x|), exactly
    quantum = torch.clamp(power * 2.0 ** -10, min=2.0 ** -24)
    return torch.round(x / quantum) * quantum


def _quantised(x):
    """The fp32 values that the rows x [..., hd] stand for once they are in the cache (64 bits next to the borders)."""
    g = x.double().unflatten(-1, (-1, 64))
    m = _to_half(g.amin(-1, keepdim=True))
    d = _to_half(torch.clamp((g.amax(-1, keepdim=True) - m) / 15, min=0))
    code = torch.where(d > 0, torch.round((g - m) / d).clamp(0, 15), torch.zeros_like(g))
    return (m + d * code).flatten(-2).float()


def _rotated(x, pos, rope_type, theta):
    """RoPE of the head rows x [n][heads][hd] at positions pos [n]: the angle is the fp32 product of position and fp32
    frequency, everything behind it is exact, the result is rounded to fp32."""
    hd = x.shape[-1]
    e = (-2.0 * torch.arange(hd // 2, device=x.device, dtype=torch.float32)) / hd
    freq = torch.pow(torch.tensor(theta, dtype=torch.float32).double().to(x.device), e.double()).float()
    ang = (pos.float()[:, None] * freq).double()[:, None]
    c, s = torch.cos(ang), torch.sin(ang)
    x = x.double()
    a, b = (x[..., : hd // 2], x[..., hd // 2:]) if rope_type == ROPE_NEOX else (x[..., 0::2], x[..., 1::2])
    a, b = a * c - b * s, a * s + b * c
    y = torch.cat((a, b), -1) if rope_type == ROPE_NEOX else torch.stack((a, b), -1).flatten(-2)
    return y.float()


def _plain(s):
    c = s["case"]
    op, hd, n_kv = c["op"], c["head_dim"], c["n_kv"]
    if op == "load":
        k, v = _values(s["cache"], hd)
        at = slice(c["row"], c["row"] + c["rows"])
        return {"k": k[:, at].half(), "v": v[:, at].half()}
    if op == "store":
        return {n: _quantised(s[n]).transpose(0, 1).half() for n in ("k", "v")}
    if op == "roll":
        n_keep, shift, n_ctx = c["n_keep"], c["shift"], c["n_ctx"]
        got = {}
        for n, x in zip(("k", "v"), _values(s["shared"], hd)):
            x = x[:, :n_ctx]
            got[n] = torch.cat((x[:, :n_keep], x[:, n_keep + shift:], torch.zeros_like(x[:, :shift])), 1).half()
        return got
    scale, group = 1.0 / math.sqrt(hd), c["n_head"] // n_kv
    k, v = _values(s["cache"], hd)
    if op == "decode":
        q = _rotated(s["q"][None], s["pos"], c["rope_type"], c["theta"])[0]
        n = c["length"]
        got = {}
        if c["append"]:
            kn = _quantised(_rotated(s["k"][None], s["pos"], c["rope_type"], c["theta"])[0])
            vn = _quantised(s["v"])
            k, v = torch.cat((k[:, : n - 1], kn[:, None]), 1), torch.cat((v[:, : n - 1], vn[:, None]), 1)
            got = {"k": kn[:, None].half(), "v": vn[:, None].half()}
        score = torch.matmul(q.view(n_kv, group, hd), k[:, :n].transpose(1, 2)) * scale
        p = torch.exp(score - score.amax(-1, keepdim=True))
        out = torch.matmul(p, v[:, :n]) / p.sum(-1, keepdim=True)
        return {"out": out.view(c["n_head"], hd), **got}
    b, past = c["batch"], c["n_past"]
    pos = torch.arange(past, past + b, device="cuda")
    q = _rotated(s["q"], pos, c["rope_type"], c["theta"])
    kn = _quantised(_rotated(s["k"], pos, c["rope_type"], c["theta"])).transpose(0, 1)
    vn = _quantised(s["v"]).transpose(0, 1)
    k, v = torch.cat((k[:, :past], kn), 1), torch.cat((v[:, :past], vn), 1)
    # [n_kv][group * b][hd] x [n_kv][hd][rows]
    score = torch.matmul(q.view(b, n_kv, group, hd).permute(1, 2, 0, 3).reshape(n_kv, group * b, hd), k.transpose(1, 2)) * scale
    unseen = torch.arange(past + b, device="cuda")[None] > pos[:, None]
    score = score.view(n_kv, group, b, past + b).masked_fill(unseen, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.matmul(p.view(n_kv, group * b, past + b), v).view(n_kv, group, b, hd) / p.sum(-1, keepdim=True)
    return {"out": out.permute(2, 0, 1, 3).reshape(b, c["n_head"], hd).half(), "k": kn.half(), "v": vn.half()}


# ---------------------------------------------------------------------------------------------------------- the library
_ops = None


def _library():
    global _ops
    if _ops is None:
        from orin_llm_b200 import ops
        ops.init(torch.cuda.current_device())
        _ops = ops
    return _ops


def _own(s):
    ops = _library()
    c = s["case"]
    op, hd, n_kv, n_ctx, cache = c["op"], c["head_dim"], c["n_kv"], s["n_ctx"], s["cache"]
    kh, vh = s["kh"], s["vh"]
    back = {"k": kh, "v": vh}
    if op == "load":
        ops.kv_load_q4(cache, kh, vh, n_kv, hd, n_ctx, c["row"], c["rows"])
        return back
    if op == "store":
        ops.kv_store_q4_batch(cache, s["k"], s["v"], n_kv, hd, n_ctx, c["pos"], c["batch"])
        ops.kv_load_q4(cache, kh, vh, n_kv, hd, n_ctx, c["pos"], c["batch"])
        return back
    if op == "roll":
        cache.copy_(s["shared"])
        ops.kv_shift_q4(cache, c["n_layer"], n_kv, hd, n_ctx, c["n_keep"], c["shift"])
        ops.kv_load_q4(cache, kh, vh, c["n_layer"] * n_kv, hd, n_ctx, 0, n_ctx)
        return back
    rope = (c["rope_type"], hd, c["theta"], None)
    scale = 1.0 / math.sqrt(hd)
    if op == "decode":
        fuse = ops.FUSE_ALL if c["append"] else ops.FUSE_ROPE_Q
        ops.attn_decode_q4(s["q"], s["k"], s["v"], cache, s["out"], c["n_head"], n_kv, hd, n_ctx, s["pos"], scale, fuse, rope)
        if not c["append"]:
            return {"out": s["out"]}
        ops.kv_load_q4(cache, kh, vh, n_kv, hd, n_ctx, c["length"] - 1, 1)
        return {"out": s["out"], **back}
    ops.attn_prefill_q4(s["q"], s["k"], s["v"], cache, s["out"], c["n_head"], n_kv, hd, n_ctx, c["n_past"], c["batch"], scale,
                        ops.FUSE_ALL, rope)
    ops.kv_load_q4(cache, kh, vh, n_kv, hd, n_ctx, c["n_past"], c["batch"])
    return {"out": s["out"], **back}


def run(s):
    return _own(s) if own else _plain(s)


# ---------------------------------------------------------------------------------------------------------- 64 bits

def _exact_rows(cache, hd, which):
    """float64 [heads][16 * blocks][hd] of K (which = 0) or V (1), read code by code from the format's addresses."""
    ng = hd // 64
    row, dim = torch.meshgrid(torch.arange(16), torch.arange(hd), indexing="ij")
    if which == 0:
        i, t, e = dim // 32, dim % 32 // 8, dim % 8
        byte = row * (hd // 2) + 4 * (t * (hd // 32) + i) + e // 2
    else:
        j, r = dim // 16, dim % 16 // 2
        byte = 8 * hd + (j // 4) * 512 + (4 * r + row % 8 // 2) * 16 + (j % 4) * 4 + 2 * (row % 2) + row // 8
    byte, odd = byte.reshape(-1).cuda(), (dim % 2 == 1).reshape(-1).cuda()
    raw = cache[..., byte].to(torch.int16)
    code = torch.where(odd, raw >> 4, raw & 15).double().view(*cache.shape[:2], 16, ng, 64)
    at = 16 * hd + which * 64 * ng
    sc = cache[..., at: at + 64 * ng].to(torch.int32).view(*cache.shape[:2], 16, ng, 2, 2)
    sc = (sc[..., 0] | (sc[..., 1] << 8)).to(torch.int16).view(torch.float16).double()
    return (sc[..., 0:1] * code + sc[..., 1:2]).reshape(cache.shape[0], -1, hd)


def _exact_quantised(x):
    """Group by group in float64; the two fp16 numbers of a group by numpy's conversion, which rounds once."""
    g = x.double().reshape(*x.shape[:-1], x.shape[-1] // 64, 64)

    def fp16(v):
        return torch.from_numpy(v.cpu().numpy().astype(np.float16).astype(np.float64)).to(v.device)

    low = fp16(g.min(-1).values)
    step = fp16(((g.max(-1).values - low) / 15).clamp(min=0))
    n = ((g - low[..., None]) / step[..., None].clamp(min=2.0 ** -24)).round().clamp(0, 15)
    n = n * (step[..., None] > 0)
    return (low[..., None] + step[..., None] * n).reshape(x.shape)


def _exact_rope(x, pos, rope_type, theta):
    hd = x.shape[-1]
    half = hd // 2
    out = x.double().clone()
    p = pos.to(torch.float32)
    for i in range(half):
        e = torch.tensor(-2.0 * i, dtype=torch.float32) / hd
        f = torch.tensor(float(torch.tensor(theta, dtype=torch.float32)) ** float(e), dtype=torch.float64).float().cuda()
        ang = (p * f).double()[:, None]
        a, b = (i, i + half) if rope_type == ROPE_NEOX else (2 * i, 2 * i + 1)
        u, v = x[..., a].double(), x[..., b].double()
        out[..., a] = u * ang.cos() - v * ang.sin()
        out[..., b] = u * ang.sin() + v * ang.cos()
    return out


def exact(c, seed):
    s = prepare(c, seed)
    op, hd, n_kv = c["op"], c["head_dim"], c["n_kv"]
    if op == "store":
        return {n: _exact_quantised(s[n]).transpose(0, 1) for n in ("k", "v")}
    if op == "load":
        return {n: _exact_rows(s["cache"], hd, w)[:, c["row"]: c["row"] + c["rows"]] for w, n in enumerate(("k", "v"))}
    if op == "roll":
        got = {}
        for w, n in enumerate(("k", "v")):
            x = _exact_rows(s["shared"], hd, w)[:, : c["n_ctx"]]
            y = torch.zeros_like(x)
            y[:, : c["n_keep"]] = x[:, : c["n_keep"]]
            y[:, c["n_keep"]: c["n_ctx"] - c["shift"]] = x[:, c["n_keep"] + c["shift"]:]
            got[n] = y
        return got
    K, V = _exact_rows(s["cache"], hd, 0), _exact_rows(s["cache"], hd, 1)
    group = c["n_head"] // n_kv
    first = c["n_past"] if op == "prefill" else c["length"] - 1
    q = s["q"] if op == "prefill" else s["q"][None]
    b = q.shape[0]
    pos = torch.arange(first, first + b, device="cuda")
    # a query is held in fp32 once it is rotated, and so is a key before it is quantised
    q = _exact_rope(q, pos, c["rope_type"], c["theta"])
    got = {}
    if op == "prefill" or c["append"]:
        k, v = (s["k"], s["v"]) if op == "prefill" else (s["k"][None], s["v"][None])
        k = _exact_quantised(_exact_rope(k, pos, c["rope_type"], c["theta"]).float()).transpose(0, 1)
        v = _exact_quantised(v).transpose(0, 1)
        K[:, first: first + b], V[:, first: first + b] = k, v
        got = {"k": k, "v": v}
    out = torch.zeros(b, c["n_head"], hd, dtype=torch.float64, device="cuda")
    for h in range(c["n_head"]):
        Kh, Vh = K[h // group, : first + b], V[h // group, : first + b]
        z = q[:, h] @ Kh.T / math.sqrt(hd)
        z = torch.where(torch.arange(first + b, device="cuda")[None] <= pos[:, None], z, torch.full_like(z, -math.inf))
        out[:, h] = torch.softmax(z, -1) @ Vh
    return {"out": out if op == "prefill" else out[0], **got}
