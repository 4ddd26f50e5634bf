"""The operators around an 8-bit paged K/V cache, as cases that can be timed and checked.

Three uses, each one pass through the public entry points (kvcache_amd.ops):

  rope    the q|k|v rows of a projection: RMSNorm of every query and key head, rotary
          position, q to its rows, k and v into the paged cache (fp16, or 8-bit codes with
          one scale per row of a head) -- qk_norm_rope_write
  round   K/V rows quantised as they are written, and read back -- write_kv_q8, read_kv
  attn    attention of a ragged batch over the paged cache: every sequence brings one new
          token or a chunk of them, already in the cache -- chunk_plan, paged_chunk_attn

`own` says whether run() computes an operator from elementary torch operations (False) or
calls the library (True).  Lengths belong to the case (so that its bytes are known), values
and block order to the seed.

Definitions.  A row x of one token and head (D values) is held as codes c and a scale s:
int8: s = max|x| / 127, c = round(x / s); e4m3: s = max|x| / 448, c = e4m3(x / s); both
round half to even.  The scales of a pool lie beside it as [block, kv head, slot, {k, v}].
Attention: query i of a chunk of n, the sequence then holding t tokens, sits at position
p = t - n + i and sees keys max(0, p - window + 1) .. p (window 0: from 0 on); the score
z = scale q.k becomes cap tanh(z / cap) where a cap is given.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
EPS, THETA = 1e-6, 1e6


# ---- the cases ---------------------------------------------------------------------------

def listed():
    return [
        # decode step of 32 running sequences: their new rows go into an fp8 cache
        {"name": "rope-step-32-14q2kv-e4m3", "kind": "rope", "rows": 32, "hq": 14, "hkv": 2, "d": 64, "block": 16,
         "cache": "e4m3", "max_pos": 32768},
        # stacked prompts of 8192 tokens, wide heads, straight into the fp8 cache
        {"name": "rope-prompt-8192-32q8kv-e4m3", "kind": "rope", "rows": 8192, "hq": 32, "hkv": 8, "d": 128,
         "block": 16, "cache": "e4m3", "max_pos": 131072},
        # an odd number of rows, heads that are not grouped, int8, read back (a cache inspected or moved)
        {"name": "rope-1531-8q8kv-i8", "kind": "rope", "rows": 1531, "hq": 8, "hkv": 8, "d": 64, "block": 16,
         "cache": "i8", "max_pos": 4096},
        # the rows of one step quantised and read back: the smallest call
        {"name": "round-96-2kv-i8", "kind": "round", "rows": 96, "hkv": 2, "d": 64, "block": 16, "cache": "i8"},
        # a long context's rows quantised as they arrive from elsewhere, and read back
        {"name": "round-40009-8kv-d128-i8", "kind": "round", "rows": 40009, "hkv": 8, "d": 128, "block": 16,
         "cache": "i8"},
        # one request at a time: one new token behind about a thousand
        {"name": "one-1000-14q2kv-i8", "kind": "attn", "cache": "i8", "n": 1, "mode": "one", "q_lo": 1, "q_hi": 1,
         "lo": 1000, "hi": 1000, "hq": 14, "hkv": 2, "d": 64, "block": 16, "window": 0, "cap": 0.0, "lens_seed": 1},
        # a wide decode batch, lengths over two decades, grouped wide heads
        {"name": "decode-200-32q8kv-d128-i8", "kind": "attn", "cache": "i8", "n": 200, "mode": "one", "q_lo": 1,
         "q_hi": 1, "lo": 32, "hi": 4096, "hq": 32, "hkv": 8, "d": 128, "block": 16, "window": 0, "cap": 0.0,
         "lens_seed": 7},
        # a decode batch of heads that are not grouped
        {"name": "decode-128-8q8kv-e4m3", "kind": "attn", "cache": "e4m3", "n": 128, "mode": "one", "q_lo": 1,
         "q_hi": 1, "lo": 16, "hi": 2048, "hq": 8, "hkv": 8, "d": 64, "block": 16, "window": 0, "cap": 0.0,
         "lens_seed": 12345},
        # few long contexts
        {"name": "decode-4-long-14q2kv-e4m3", "kind": "attn", "cache": "e4m3", "n": 4, "mode": "one", "q_lo": 1,
         "q_hi": 1, "lo": 8000, "hi": 32768, "hq": 14, "hkv": 2, "d": 64, "block": 16, "window": 0, "cap": 0.0,
         "lens_seed": 3},
        # a continuous-batching step: most sequences decode, some bring a chunk of their prompt
        {"name": "mixed-48-14q2kv-i8", "kind": "attn", "cache": "i8", "n": 48, "mode": "mixed", "q_lo": 2,
         "q_hi": 300, "lo": 32, "hi": 4096, "hq": 14, "hkv": 2, "d": 64, "block": 16, "window": 0, "cap": 0.0,
         "lens_seed": 11},
        # a piece of a long prompt behind 6000 tokens that are already cached
        {"name": "chunk-2000-at-6000-32q8kv-d128-i8", "kind": "attn", "cache": "i8", "n": 1, "mode": "all",
         "q_lo": 2000, "q_hi": 2000, "lo": 6000, "hi": 6000, "hq": 32, "hkv": 8, "d": 128, "block": 16, "window": 0,
         "cap": 0.0, "lens_seed": 5},
        # chunks of four long prompts with capped scores and a sliding window, fp16 cache
        {"name": "chunk-4x700-window-cap-f16", "kind": "attn", "cache": "f16", "n": 4, "mode": "all", "q_lo": 500,
         "q_hi": 900, "lo": 3500, "hi": 9000, "hq": 16, "hkv": 4, "d": 128, "block": 16, "window": 1024, "cap": 30.0,
         "lens_seed": 9},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


_HEADS = [(14, 2, 64), (8, 8, 64), (16, 4, 64), (12, 12, 64), (32, 8, 128), (16, 16, 128), (16, 4, 128), (8, 1, 128)]


def _drawn(rng):
    kind = rng.choice(["rope", "rope", "round", "attn", "attn", "attn", "attn"])
    hq, hkv, d = rng.choice(_HEADS)
    block = rng.choice([16, 16, 16, 32, 64])
    if kind == "rope":
        return {"kind": kind, "rows": _log_int(rng, 1, 8192), "hq": hq, "hkv": hkv, "d": d, "block": block,
                "cache": rng.choice(["i8", "e4m3", "f16"]), "max_pos": rng.choice([2048, 32768, 1 << 20])}
    if kind == "round":
        return {"kind": kind, "rows": _log_int(rng, 1, 40000), "hkv": hkv, "d": d, "block": block,
                "cache": rng.choice(["i8", "e4m3"])}
    mode = rng.choice(["one", "one", "mixed", "all"])
    c = {"kind": kind, "cache": rng.choice(["i8", "i8", "e4m3", "e4m3", "f16"]), "n": 1, "mode": mode, "q_lo": 1,
         "q_hi": 1, "lo": 1, "hi": 1, "hq": hq, "hkv": hkv, "d": d, "block": block,
         "window": rng.choice([0, 0, 0, _log_int(rng, 100, 4096)]), "cap": rng.choice([0.0, 0.0, 0.0, 20.0, 50.0]),
         "lens_seed": rng.randrange(1, 1 << 20)}
    c["hi"] = _log_int(rng, 64, 32768)
    c["lo"] = _log_int(rng, 1, c["hi"])
    if mode == "one":
        c["n"] = _log_int(rng, 1, 200)
    elif mode == "mixed":
        c["n"], c["q_lo"], c["q_hi"] = _log_int(rng, 2, 64), 1, _log_int(rng, 2, 600)
    else:
        c["n"], c["q_hi"] = _log_int(rng, 1, 16), _log_int(rng, 1, 2500)
        c["q_lo"] = _log_int(rng, 1, c["q_hi"])
    return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng: random.Random):
    most = max(_cost(c) for c in listed())
    while True:
        c = _drawn(rng)
        # (the plain form's padded scores and keys have to stay within a few GB)
        if c["kind"] == "attn":
            q, t = _lens(c)
            if len(q) * c["hq"] * int(q.max()) * int(t.max()) > 8e8 or len(q) * c["hkv"] * c["d"] * int(t.max()) > 1.2e9:
                continue
        if _cost(c) <= most:
            return c


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, std=1.0):
    t = torch.empty(shape, device=DEV, dtype=torch.float16)
    t.normal_(0.0, std, generator=g)
    return t


def _lens(case):
    """New tokens and tokens altogether (the new ones included) of every sequence."""
    r = np.random.default_rng(case["lens_seed"])
    n = case["n"]

    def log_ints(lo, hi):
        return np.clip(np.exp(r.uniform(math.log(lo), math.log(hi + 1), n)).astype(np.int64), lo, hi)

    before, q = log_ints(case["lo"], case["hi"]), log_ints(case["q_lo"], case["q_hi"])
    if case["mode"] == "mixed":
        q = np.where(r.random(n) < 0.25, q, 1)
    return q.astype(np.int32), (before + q).astype(np.int32)


_CODES = {"i8": torch.int8, "e4m3": torch.uint8, "f16": torch.float16}


def _pools(case, blocks):
    shape = (blocks, case["hkv"], case["block"], case["d"])
    p = {"k_pool": torch.zeros(shape, dtype=_CODES[case["cache"]], device=DEV),
         "v_pool": torch.zeros(shape, dtype=_CODES[case["cache"]], device=DEV)}
    if case["cache"] != "f16":
        p["scales"] = torch.zeros(shape[:3] + (2,), dtype=torch.float32, device=DEV)
    return p


def _inputs(case, seed):
    g, kind, d, b = _gen(seed), case["kind"], case["d"], case["block"]
    hkv = case["hkv"]
    if kind in ("rope", "round"):
        m = case["rows"]
        nb = (m + b - 1) // b + 2
        s = {"nb": nb}
        # rows in the order of their sequences' tokens, blocks anywhere in the pool
        at = torch.arange(m, device=DEV)
        order = torch.randperm(nb, device=DEV, generator=g)
        s["slots"] = (order[at // b] * b + at % b).to(torch.int32)
        if kind == "rope":
            s["qkv"] = _normal(g, (m, (case["hq"] + 2 * hkv) * d), 0.7)
            s["q_norm"], s["k_norm"] = 1 + _normal(g, (d,), 0.1), 1 + _normal(g, (d,), 0.1)
            first = torch.randint(0, case["max_pos"], (1,), device=DEV, generator=g)
            step = torch.randint(0, case["max_pos"], (m,), device=DEV, generator=g)
            s["pos"] = (step if m <= 64 else first + at).to(torch.int32)
        else:
            size = torch.exp(0.5 * torch.randn((2, m, hkv, 1), device=DEV, generator=g))
            s["k"], s["v"] = (_normal(g, (m, hkv, d)) * size[0]).half(), (_normal(g, (m, hkv, d)) * size[1]).half()
        return s
    q, t = _lens(case)
    nblk = (t + b - 1) // b
    off = np.concatenate([[0], np.cumsum(nblk)]).astype(np.int32)
    nb = int(off[-1])
    s = {"table": torch.randperm(nb, device=DEV, generator=g).to(torch.int32), "off": off, "q_lens": q, "kv_lens": t}
    s["q"] = _normal(g, (int(q.sum()), case["hq"], d))
    shape = (nb, hkv, b, d)
    if case["cache"] == "f16":
        s["k_pool"], s["v_pool"] = _normal(g, shape), _normal(g, shape)
    else:
        # rows whose sizes differ by token, as those of a trained model do
        for i, name in enumerate(("k_pool", "v_pool")):
            size = torch.exp(0.4 * torch.randn(shape[:3] + (1,), device=DEV, generator=g))
            codes, sc = _quantise(_normal(g, shape).float() * size, case["cache"])
            s[name] = codes
            s.setdefault("scales", torch.empty(shape[:3] + (2,), device=DEV))[..., i] = sc
    # the sequences side by side: table and query rows padded to the longest (the plain form's layout)
    n, mb, mq = len(q), int(nblk.max()), int(q.max())
    tab = np.minimum(off[:-1, None] + np.minimum(np.arange(mb)[None], nblk[:, None] - 1), nb - 1)
    s["tab_pad"] = s["table"][torch.from_numpy(tab.astype(np.int64)).to(DEV)].long()
    row0 = np.concatenate([[0], np.cumsum(q)[:-1]])
    i = np.arange(mq)[None]
    s["row_pad"] = torch.from_numpy((row0[:, None] + np.minimum(i, q[:, None] - 1)).astype(np.int64)).to(DEV)
    s["pos_pad"] = torch.from_numpy((t[:, None] - q[:, None] + np.minimum(i, q[:, None] - 1)).astype(np.int64)).to(DEV)
    s["row_of"] = torch.from_numpy(np.flatnonzero((i < q[:, None]).reshape(-1)).astype(np.int64)).to(DEV)
    s["n"] = n
    return s


def _address(s):
    """The addresses a C caller would hold."""
    s["p"] = {k: t.data_ptr() for k, t in s.items() if isinstance(t, torch.Tensor)}
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if kind in ("rope", "round"):
        s.update(_pools(case, s["nb"]))
        m, d = case["rows"], case["d"]
        if kind == "rope":
            s["q_out"] = torch.zeros((m, case["hq"], d), dtype=torch.float16, device=DEV)
        s["k_out"] = torch.zeros((m, case["hkv"], d), dtype=torch.float16, device=DEV)
        s["v_out"] = torch.zeros_like(s["k_out"])
    else:
        s["scale"] = case["d"] ** -0.5
        s["out"] = torch.zeros_like(s["q"])
        if own:
            # the step's plan and workspace: the scheduler makes them once, every layer's launch uses them
            from kvcache_amd import ops
            work_list, units, tiles, records = ops.chunk_plan(s["q_lens"], s["kv_lens"], case["hq"], case["hkv"],
                                                              case["d"], case["block"], kv_dtype=_kv_dtype(case),
                                                              window=case["window"], tab_off=s["off"])
            s["plan"] = torch.from_numpy(np.ascontiguousarray(work_list)).to(DEV)
            s["units"], s["tiles"], s["records"] = units, tiles, records
            size = ops.chunk_workspace_size(case["hq"], case["hkv"], case["d"], records)
            s["ws"] = torch.zeros(max(size, 256), dtype=torch.uint8, device=DEV)
    return _address(s)


def _kv_dtype(case):
    from kvcache_amd import _native
    return {"f16": _native.KVC_F16, "i8": _native.KVC_I8, "e4m3": _native.KVC_E4M3}[case["cache"]]


# ---- one pass ----------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return {"rope": _own_rope, "round": _own_round, "attn": _own_attn}[c["kind"]](c, s)
    return {"rope": _plain_rope, "round": _plain_round, "attn": _plain_attn}[c["kind"]](c, s)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _written(c, s, **more):
    """A pass's outputs: the cache as the values its codes stand for, and the scales."""
    if c["cache"] == "f16":
        return {**more, "k": s["k_pool"], "v": s["v_pool"]}
    if c["cache"] == "e4m3" and c["kind"] == "rope":
        return {**more, "k": s["k_pool"].view(torch.float8_e4m3fn), "v": s["v_pool"].view(torch.float8_e4m3fn),
                "scales": s["scales"]}
    return {**more, "k": s["k_out"], "v": s["v_out"], "scales": s["scales"]}


def _own_read(c, s):
    from kvcache_amd import ops
    p = s["p"]
    ops.read_kv(p["k_out"], p["v_out"], p["k_pool"], p["v_pool"], p["scales"], p["slots"], c["rows"], c["hkv"],
                c["d"], c["block"], kv_dtype=_kv_dtype(c), stream=_stream())


def _own_rope(c, s):
    from kvcache_amd import ops
    p = s["p"]
    ops.qk_norm_rope_write(p["q_out"], p["k_pool"], p["v_pool"], p.get("scales"), p["qkv"], p["pos"], p["slots"],
                           c["rows"], c["hq"], c["hkv"], c["d"], c["block"], THETA, q_norm=p["q_norm"],
                           k_norm=p["k_norm"], eps=EPS, kv_dtype=_kv_dtype(c), stream=_stream())
    if c["cache"] == "i8":
        _own_read(c, s)
    return _written(c, s, q=s["q_out"])


def _own_round(c, s):
    from kvcache_amd import ops
    p = s["p"]
    ops.write_kv_q8(p["k"], p["v"], p["k_pool"], p["v_pool"], p["scales"], p["slots"], c["rows"], c["hkv"], c["d"],
                    c["block"], kv_dtype=_kv_dtype(c), stream=_stream())
    _own_read(c, s)
    return _written(c, s)


def _own_attn(c, s):
    from kvcache_amd import ops
    p = s["p"]
    ops.paged_chunk_attn(p["q"], p["out"], p["k_pool"], p["v_pool"], p.get("scales"), p["table"], len(s["table"]),
                         p["plan"], s["units"], s["tiles"], s["records"], len(s["q"]), c["hq"], c["hkv"], c["d"],
                         c["block"], s["scale"], kv_dtype=_kv_dtype(c), softcap=c["cap"], window=c["window"],
                         workspace=(p["ws"], s["ws"].numel()), stream=_stream())
    return s["out"]


# ---- the same from elementary operations ---------------------------------------------------

def _quantise(x, cache):
    """Codes and scales of fp32 rows [..., D]."""
    s = x.abs().amax(-1) / (127.0 if cache == "i8" else 448.0)
    y = x / torch.where(s > 0, s, 1.0)[..., None]
    if cache == "i8":
        return torch.round(y).to(torch.int8), s
    return y.to(torch.float8_e4m3fn).view(torch.uint8), s


def _values(codes, cache):
    if cache == "e4m3":
        codes = codes.view(torch.float8_e4m3fn)
    return codes.float()


def _plain_store(c, s, k, v):
    """fp32 rows [m, hkv, D] into the pools at their slots."""
    blk, at = torch.div(s["slots"].long(), c["block"], rounding_mode="floor"), s["slots"].long() % c["block"]
    if c["cache"] == "f16":
        s["k_pool"][blk, :, at] = k.half()
        s["v_pool"][blk, :, at] = v.half()
        return
    kc, ks = _quantise(k, c["cache"])
    vc, vs = _quantise(v, c["cache"])
    s["k_pool"][blk, :, at] = kc
    s["v_pool"][blk, :, at] = vc
    s["scales"][blk, :, at] = torch.stack([ks, vs], -1)


def _plain_read(c, s):
    blk, at = torch.div(s["slots"].long(), c["block"], rounding_mode="floor"), s["slots"].long() % c["block"]
    sc = s["scales"][blk, :, at]
    s["k_out"].copy_(_values(s["k_pool"][blk, :, at], c["cache"]) * sc[..., :1])
    s["v_out"].copy_(_values(s["v_pool"][blk, :, at], c["cache"]) * sc[..., 1:])


def _plain_rope(c, s):
    m, hq, hkv, d = c["rows"], c["hq"], c["hkv"], c["d"]
    x = s["qkv"].view(m, hq + 2 * hkv, d).float()
    # angles in 64 bits: a far position times a frequency has too many turns for 32
    turn = torch.exp2(torch.arange(d // 2, device=DEV, dtype=torch.float64) * (-2.0 * math.log2(THETA) / d))
    ang = s["pos"].double()[:, None] * turn
    co, si = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]

    def normed(y, w):
        return y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()

    def turned(y):
        a, b = y[..., :d // 2], y[..., d // 2:]
        return torch.cat([a * co - b * si, b * co + a * si], -1)

    s["q_out"].copy_(turned(normed(x[:, :hq], s["q_norm"])))
    _plain_store(c, s, turned(normed(x[:, hq:hq + hkv], s["k_norm"])), x[:, hq + hkv:])
    if c["cache"] == "i8":
        _plain_read(c, s)
    return _written(c, s, q=s["q_out"])


def _plain_round(c, s):
    _plain_store(c, s, s["k"].float(), s["v"].float())
    _plain_read(c, s)
    return _written(c, s)


def _plain_attn(c, s):
    n, hq, hkv, d, b = s["n"], c["hq"], c["hkv"], c["d"], c["block"]
    tab, rows, pos = s["tab_pad"], s["row_pad"], s["pos_pad"]
    mb, mq = tab.shape[1], rows.shape[1]

    def cached(name, i):
        x = s[name][tab]                                        # [n, mb, hkv, b, d]
        x = x.float() if c["cache"] == "f16" else _values(x, c["cache"]) * s["scales"][..., i][tab][..., None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, hkv, mb * b, d)

    q = s["q"][rows].float().view(n, mq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    z = torch.matmul(q, cached("k_pool", 0).transpose(2, 3).contiguous()) * s["scale"]
    if c["cap"]:
        z = c["cap"] * torch.tanh(z / c["cap"])
    key = torch.arange(mb * b, device=DEV)
    seen = key <= pos[:, :, None]
    if c["window"]:
        seen &= key > pos[:, :, None] - c["window"]
    z = z.view(n, hkv, hq // hkv, mq, mb * b).masked_fill_(~seen[:, None, None], -math.inf)
    e = torch.exp(z - z.amax(-1, keepdim=True)).view(n, hkv, -1, mb * b)
    out = torch.matmul(e, cached("v_pool", 1)) / e.sum(-1, keepdim=True)
    out = out.view(n, hkv, hq // hkv, mq, d).permute(0, 3, 1, 2, 4).reshape(n * mq, hq, d)
    s["out"].copy_(out[s["row_of"]])
    return s["out"]


# ---- what a pass cannot do without --------------------------------------------------------

def work(case):
    c, d, hkv = case, case["d"], case["hkv"]
    code, sc = (2, 0) if c["cache"] == "f16" else (1, 8)  # bytes of a cached value; of a token's two scales
    if c["kind"] == "rope":
        m, hq = c["rows"], c["hq"]
        moved = m * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + hkv * (2 * d * code + sc) + 8) + 2 * d * 2
        if c["cache"] == "i8":  # read back: the codes and scales, and the rows they stand for
            moved += m * hkv * (2 * d * code + sc + 2 * d * 2)
        return {"bytes": moved, "flops": m * (hq + hkv) * d * 8}
    if c["kind"] == "round":
        m = c["rows"]
        return {"bytes": m * (hkv * (2 * d * 2 + 2 * (2 * d * code + sc) + 2 * d * 2) + 4), "flops": m * hkv * d * 8}
    q, t = _lens(c)
    q, t = q.astype(np.int64), t.astype(np.int64)
    p0, w = t - q, c["window"] or 1 << 40
    pairs = sum(int(np.minimum(np.arange(a, b) + 1, w).sum()) for a, b in zip(p0, t))
    keys = int((t - np.maximum(0, p0 - w + 1)).sum())
    return {"bytes": keys * hkv * (2 * d * code + sc) + 2 * int(q.sum()) * c["hq"] * d * 2,
            "flops": 4 * pairs * c["hq"] * d}


# ---- the same in 64 bits ------------------------------------------------------------------

def _e4m3_64(y):
    """Doubles rounded to the nearest value of e4m3, half to even."""
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0)
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def _held64(x, cache):
    """What the cache holds of rows x: (codes as values, scale)."""
    if cache == "f16":
        return x, None
    top = 127.0 if cache == "i8" else 448.0
    sc = x.abs().amax(-1, keepdim=True) / top
    y = torch.where(sc > 0, x / sc.clamp_min(1e-300), 0.0)
    return (torch.round(y) if cache == "i8" else _e4m3_64(y)), sc


def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    hkv, d, b = c["hkv"], c["d"], c["block"]
    if c["kind"] in ("rope", "round"):
        m, nb, slots = c["rows"], s["nb"], s["slots"].long()
        out = {}
        if c["kind"] == "rope":
            hq = c["hq"]
            x = s["qkv"].double().reshape(m, hq + 2 * hkv, d)

            def head(y, w):
                y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / d + EPS) * w.double()
                t = torch.arange(d // 2, device=DEV, dtype=torch.float64)
                z = torch.polar(torch.ones((m, 1, d // 2), dtype=torch.float64, device=DEV),
                                (s["pos"].double()[:, None] * THETA ** (-2.0 * t / d))[:, None])
                z = z * torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous())
                return torch.cat([z.real, z.imag], -1)

            out["q"] = head(x[:, :hq], s["q_norm"])
            k, v = head(x[:, hq:hq + hkv], s["k_norm"]), x[:, hq + hkv:]
        else:
            k, v = s["k"].double(), s["v"].double()
        (kc, ks), (vc, vs) = _held64(k, c["cache"]), _held64(v, c["cache"])

        def pool(rows):
            y = torch.zeros((nb * b,) + rows.shape[1:], dtype=torch.float64, device=DEV)
            y[slots] = rows
            return y.reshape((nb, b) + rows.shape[1:]).transpose(1, 2).contiguous()

        if c["cache"] != "f16":
            out["scales"] = pool(torch.cat([ks, vs], -1))
        if c["cache"] == "f16" or (c["cache"] == "e4m3" and c["kind"] == "rope"):
            out["k"], out["v"] = pool(kc), pool(vc)
        else:
            out["k"], out["v"] = kc * ks, vc * vs
        return out
    res, row = [], 0
    for i, (n, t) in enumerate(zip(s["q_lens"].tolist(), s["kv_lens"].tolist())):
        blocks = s["table"][s["off"][i]:s["off"][i + 1]].long()
        first = max(0, t - n - c["window"] + 1) // b if c["window"] else 0  # blocks before it hold no key of these
        blocks = blocks[first:]

        def tokens(name, j):
            x = s[name][blocks]
            if c["cache"] == "e4m3":
                x = x.view(torch.float8_e4m3fn).float()
            x = x.double()
            if c["cache"] != "f16":
                x = x * s["scales"][blocks][..., j:j + 1].double()
            return x.transpose(1, 2).reshape(-1, hkv, d)[:t - first * b]

        k, v = tokens("k_pool", 0), tokens("v_pool", 1)
        at = torch.arange(first * b, t, device=DEV)[None]
        p = torch.arange(t - n, t, device=DEV)[:, None]
        hide = at > p if not c["window"] else (at > p) | (at <= p - c["window"])
        g = c["hq"] // hkv
        q = s["q"][row:row + n].double()
        y = torch.empty((n, c["hq"], d), dtype=torch.float64, device=DEV)
        for h in range(c["hq"]):
            z = q[:, h] @ k[:, h // g].T.contiguous() * d ** -0.5
            if c["cap"]:
                z = c["cap"] * torch.tanh(z / c["cap"])
            y[:, h] = torch.softmax(z.masked_fill(hide, -math.inf), -1) @ v[:, h // g].contiguous()
        res.append(y)
        row += n
    return torch.cat(res)
