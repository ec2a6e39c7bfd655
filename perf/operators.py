"""The 8-bit serving operators as they are used: RMSNorm with the residual's addition and an 8-bit output, the
e4m3 matrix product with a scale for each block of 128, the append to a cache held in 8 bits with the attention
that reads it, and sampling with temperature, top-k, top-p and min-p.

Every case has a plain form (elementary torch operations) and the library's calls (``own``) on the same state.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
QMAX = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
EPS = 1e-5


def cdiv(a, b):
    return -(-a // b)


def listed():
    return [
        # the norm before a projection: one decoded token, and a long prompt of a 5120-wide model
        {"name": "norm_token", "op": "norm", "rows": 1, "dim": 8192, "dtype": "f32", "code": "e4m3", "group": 128},
        {"name": "norm_prompt", "op": "norm", "rows": 4099, "dim": 5120, "dtype": "bf16", "code": "e4m3", "group": 128},
        # projections: q|k|v of one token, down of a batch of 16, down of an odd batch, gate of a 2048-token prompt
        {"name": "gemm_token_qkv", "op": "gemm", "M": 1, "N": 10240, "K": 8192, "dtype": "f32"},
        {"name": "gemm_batch_down", "op": "gemm", "M": 16, "N": 8192, "K": 28672, "dtype": "bf16"},
        {"name": "gemm_odd_down", "op": "gemm", "M": 197, "N": 5120, "K": 13824, "dtype": "f16"},
        {"name": "gemm_prompt_gate", "op": "gemm", "M": 2048, "N": 28672, "K": 8192, "dtype": "bf16"},
        # attention of one token of one sequence (64 heads on 8), of a ragged batch, of a few long sequences,
        # and of a 2048-token piece of a prompt over what came before it (40 heads on 40)
        {"name": "attend_token", "op": "attend", "seqs": 1, "n": 1, "heads": 64, "kv_heads": 8, "D": 128, "max_seq": 2048,
         "lo": 2000, "hi": 2000, "dtype": "f32", "code": "int8", "block": 64},
        {"name": "attend_batch", "op": "attend", "seqs": 16, "n": 1, "heads": 64, "kv_heads": 8, "D": 128, "max_seq": 8192,
         "lo": 301, "hi": 8100, "dtype": "bf16", "code": "e4m3", "block": 64},
        {"name": "attend_long", "op": "attend", "seqs": 3, "n": 1, "heads": 32, "kv_heads": 8, "D": 128, "max_seq": 65536,
         "lo": 40001, "hi": 65000, "dtype": "f16", "code": "int8", "block": 128},
        {"name": "attend_prompt", "op": "attend", "seqs": 1, "n": 2048, "heads": 40, "kv_heads": 40, "D": 128,
         "max_seq": 8192, "lo": 2001, "hi": 2001, "dtype": "bf16", "code": "e4m3", "block": 64},
        # the next token: one row of a 32,000-entry vocabulary, and a batch over a vocabulary of 100,277
        {"name": "sample_token", "op": "sample", "rows": 1, "V": 32000, "dtype": "f32"},
        {"name": "sample_batch", "op": "sample", "rows": 64, "V": 100277, "dtype": "f32"},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "gemm", "attend", "attend", "sample"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        return {"op": op, "rows": log(1, 4096), "dim": log(100, 16384), "dtype": dtype,
                "code": rng.choice(["e4m3", "e4m3", "int8"]), "group": rng.choice([128, 128, 0])}
    if op == "gemm":
        M, N, K = log(1, 2048), log(64, 28672), log(128, 28672)
        while M * N * K > 2048 * 28672 * 8192:
            M = max(1, M // 2)
        return {"op": op, "M": M, "N": N, "K": K, "dtype": dtype}
    if op == "attend":
        kv_heads, D = rng.choice([1, 2, 8, 40]), rng.choice([64, 128, 128, 256])
        heads = kv_heads * (1 if kv_heads == 40 else rng.choice([1, 3, 4, 8]))
        n = rng.choice([1, 1, 1, log(2, 2048)])
        max_seq = max(log(64, 65536 if n == 1 else 8192), n + 1)
        seqs = log(1, 64 if n == 1 else 4)
        # no more than the largest listed cases: their cache, and their products and rows of scores
        while seqs > 1 and (seqs * kv_heads * max_seq * D > 3 * 8 * 65536 * 128 or seqs * heads * n * max_seq * D > 40 * 2048 * 4049 * 128):
            seqs //= 2
        while n > 1 and seqs * heads * n * max_seq * D > 40 * 2048 * 4049 * 128:
            n = max(1, n // 2)
        while seqs * kv_heads * max_seq * D > 3 * 8 * 65536 * 128:
            max_seq //= 2
        n = min(n, max_seq - 1)
        hi = max_seq - n
        return {"op": op, "seqs": seqs, "n": n, "heads": heads, "kv_heads": kv_heads, "D": D, "max_seq": max_seq,
                "lo": rng.randint(0, hi), "hi": hi, "dtype": dtype, "code": rng.choice(["int8", "e4m3"]),
                "block": rng.choice([16, 32, 64, 128])}
    rows, V = log(1, 64), log(500, 100277)
    return {"op": op, "rows": rows, "V": V, "dtype": dtype}


def past_lengths(c):
    """Tokens of each sequence before the call: spread over [lo, hi] in a fixed irregular order."""
    return [c["lo"] + int((c["hi"] - c["lo"]) * ((b * 0.6180339887 + 0.77) % 1.0)) for b in range(c["seqs"])]


# ---- inputs -------------------------------------------------------------------------------------

def blocks_of(x, block):
    """[..., n] -> [..., ceil(n / block), block], padded with zeros."""
    n = x.shape[-1]
    pad = cdiv(n, block) * block - n
    if pad:
        x = torch.nn.functional.pad(x, (0, pad))
    return x.reshape(*x.shape[:-1], -1, block)


def to_codes(v, code):
    """v (fp32, within the code's range) rounded to the nearest code, ties to even."""
    q = QMAX[code]
    if code == "int8":
        return torch.round(v).clamp(-q, q).to(torch.int8)
    return v.clamp(-q, q).to(torch.float8_e4m3fn)


def aligned_rows(codes, K):
    """Codes [rows][K] in a buffer whose rows start on 16-byte boundaries, as a user lays them out."""
    ld = cdiv(K, 16) * 16
    buf = torch.zeros(codes.shape[0], ld, dtype=torch.uint8, device="cuda")
    buf[:, :K] = codes.view(torch.uint8)
    return buf, ld


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    s = {"case": dict(c), "op": c["op"]}
    dt = DT[c["dtype"]]
    if c["op"] == "norm":
        R, D = c["rows"], c["dim"]
        x, r = randn(R, D), randn(R, D) * 2
        r[:, :: max(1, D // 7)] *= 20         # the few large channels that residual streams have
        s |= {"x": x.to(dt), "residual": r.to(dt), "weight": 1 + 0.1 * randn(D)}
        groups = cdiv(D, c["group"]) if c["group"] else 1
        s |= {"h": torch.empty(R, D, dtype=dt, device="cuda"),
              "codes": torch.empty(R, D, dtype=torch.uint8, device="cuda"),
              "scales": torch.empty(R, groups, device="cuda")}
    elif c["op"] == "gemm":
        M, N, K = c["M"], c["N"], c["K"]
        x = blocks_of(randn(M, K), 128)
        xs = x.abs().amax(-1) / 448
        x = to_codes(x / xs[..., None].clamp_min(1e-30), "e4m3").reshape(M, -1)[:, :K]
        nb, kb = cdiv(N, 128), cdiv(K, 128)
        w = randn(N, K)
        w *= 0.02
        wp = torch.zeros(nb * 128, kb * 128, device="cuda")
        wp[:N, :K] = w
        del w
        t = wp.view(nb, 128, kb, 128)
        ws = t.abs().amax((1, 3)) / 448
        t /= ws[:, None, :, None].clamp_min(1e-30)
        w = wp.to(torch.float8_e4m3fn)[:N, :K]
        del wp, t
        s["x"], s["ldx"] = aligned_rows(x.contiguous(), K)
        s["w"], s["ldw"] = aligned_rows(w.contiguous(), K)
        s |= {"xs": xs.contiguous(), "ws": ws.contiguous(), "y": torch.empty(M, N, dtype=dt, device="cuda")}
    elif c["op"] == "attend":
        B, n, H, G, D, S, T = (c[k] for k in ("seqs", "n", "heads", "kv_heads", "D", "max_seq", "block"))
        past = past_lengths(c)
        s["past_host"] = past
        s["past"] = torch.tensor(past, dtype=torch.int32, device="cuda")
        s["row_start"] = (torch.arange(B + 1, dtype=torch.int32, device="cuda") * n)
        nb = cdiv(S, T)
        for name in ("k", "v"):
            if c["code"] == "int8":
                s[name] = torch.randint(-127, 128, (B, G, S, D), generator=g, device="cuda", dtype=torch.int8)
            else:      # the codes of normal values in blocks whose largest is about 3.3
                s[name] = torch.empty(B, G, S, D, dtype=torch.float8_e4m3fn, device="cuda")
                for b in range(B):
                    s[name][b] = (torch.randn(G, S, D, generator=g, device="cuda") * 130).clamp(-448, 448).to(torch.float8_e4m3fn)
            top = 3.3 / QMAX[c["code"]]
            s[name + "_scale"] = top * (0.5 + torch.rand(B, G, nb, generator=g, device="cuda"))
            s[name + "_new"] = randn(B * n, G, D, dtype=dt)
        s["q"] = randn(B * n, H, D, dtype=dt)
        s["out"] = torch.empty(B * n, H, D, dtype=dt, device="cuda")
    else:
        R, V = c["rows"], c["V"]
        s["logits"] = (randn(R, V) * 2.5).to(dt)

        def pick(values):
            i = torch.randint(0, len(values), (R,), generator=g, device="cuda")
            return torch.tensor(values, device="cuda")[i].contiguous()

        s["temperature"] = pick([0.6, 0.8, 1.0, 1.3, 0.0])
        s["top_k"] = pick([0, 0, 40, 200, 1000]).to(torch.int32)
        s["top_p"] = pick([1.0, 0.9, 0.95, 0.5])
        s["min_p"] = pick([0.0, 0.0, 0.05, 0.1])
        s["u"] = torch.rand(R, generator=g, device="cuda")
        s["tokens"] = torch.zeros(R, dtype=torch.int32, device="cuda")
        s["probs"] = torch.zeros(R, device="cuda")
    if own:
        prepare_own(s)
    return s


# ---- the plain forms ----------------------------------------------------------------------------

def plain_norm(s):
    c = s["case"]
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"]
    group = c["group"] or c["dim"]
    t = blocks_of(y, group)
    scales = t.abs().amax(-1) / QMAX[c["code"]]
    codes = to_codes(t / torch.where(scales > 0, scales, 1.0)[..., None], c["code"])
    codes = codes.reshape(c["rows"], -1)[:, : c["dim"]]
    return norm_result(c, h.to(s["x"].dtype), codes, scales)


def norm_result(c, h, codes, scales):
    """The e4m3 codes as they are; int8 codes as the values they stand for, in half precision."""
    if c["code"] == "int8":
        group = c["group"] or c["dim"]
        codes = (codes.float() * scales.repeat_interleave(group, -1)[:, : c["dim"]]).half()
    return {"h": h, "codes": codes, "scales": scales}


def plain_gemm(s):
    c = s["case"]
    M, N, K = c["M"], c["N"], c["K"]
    x = s["x"][:, :K].view(torch.float8_e4m3fn).float() * s["xs"].repeat_interleave(128, 1)[:, :K]
    w = s["w"][:, :K].view(torch.float8_e4m3fn).float()
    w *= s["ws"].repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return (x @ w.t()).to(s["y"].dtype)


def plain_append(codes, scale, new, past, n, T, code):
    """new [B, G, n, D] to positions past.. of codes [B, G, S, D] with scale [B, G, S / T], in place."""
    B, G, S, D = codes.shape
    q = QMAX[code]
    nb = (n + T - 2) // T + 1                                                # blocks a piece can touch
    blk = past[:, None].long() // T + torch.arange(nb, device=past.device)   # [B, nb]
    pos = blk[..., None] * T + torch.arange(T, device=past.device)           # [B, nb, T]
    p0 = past[:, None, None].long()
    is_new = (pos >= p0) & (pos < p0 + n)
    live = is_new.any(-1)                                                    # [B, nb]
    held = (pos < p0) & live[..., None]
    bi = torch.arange(B, device=past.device)
    safe_blk, safe_pos = blk.clamp(max=scale.shape[2] - 1), pos.clamp(max=S - 1)
    old_scale = scale.permute(0, 2, 1)[bi[:, None], safe_blk]                # [B, nb, G]
    start = torch.where(held.any(-1)[..., None], old_scale, 0.0)
    x = new.permute(0, 2, 1, 3).float()[bi[:, None, None], (pos - p0).clamp(0, n - 1)]   # [B, nb, T, G, D]
    amax = torch.where(is_new[..., None, None], x.abs(), 0.0).amax((2, 4))   # [B, nb, G]
    grown = torch.maximum(start, amax / q)
    div = torch.where(grown > 0, grown, 1.0)[:, :, None, :, None]
    old = codes.permute(0, 2, 1, 3)[bi[:, None, None], safe_pos]             # [B, nb, T, G, D]
    kept = to_codes(old.float() * start[:, :, None, :, None] / div, code)
    same = (grown == start)[:, :, None, :, None]
    put = torch.where(is_new[..., None, None], to_codes(x / div, code).view(torch.uint8),
                      torch.where(same, old.view(torch.uint8), kept.view(torch.uint8)))
    b, j, t = torch.nonzero(is_new | held, as_tuple=True)
    codes.view(torch.uint8).permute(0, 2, 1, 3)[b, pos[b, j, t]] = put[b, j, t]
    b, j = torch.nonzero(live, as_tuple=True)
    scale.permute(0, 2, 1)[b, blk[b, j]] = grown[b, j]


def plain_attend(s):
    c = s["case"]
    B, n, H, G, D, S, T = (c[k] for k in ("seqs", "n", "heads", "kv_heads", "D", "max_seq", "block"))
    for name in ("k", "v"):
        new = s[name + "_new"].view(B, n, G, D).permute(0, 2, 1, 3)
        plain_append(s[name], s[name + "_scale"], new, s["past"], n, T, c["code"])
    L = max(s["past_host"]) + n
    k = s["k"][:, :, :L].float() * s["k_scale"].repeat_interleave(T, -1)[:, :, :L, None]
    q = s["q"].view(B, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, (H // G) * n, D).float()
    p = (q @ k.transpose(-1, -2)) * D ** -0.5
    del k
    p = p.view(B, G, H // G, n, L)
    last = s["past"][:, None] + torch.arange(n, device="cuda")              # [B, n]
    seen = torch.arange(L, device="cuda") <= last[..., None]                # [B, n, L]
    p = p.masked_fill(~seen[:, None, None], -torch.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    norm = p.sum(-1, keepdim=True)
    v = s["v"][:, :, :L].float() * s["v_scale"].repeat_interleave(T, -1)[:, :, :L, None]
    v.masked_fill_(torch.arange(L, device="cuda")[None, None, :, None] >= (s["past"] + n)[:, None, None, None], 0.0)
    o = (p.view(B, G, -1, L) @ v).view(B, G, H // G, n, D) / norm
    out = o.permute(0, 3, 1, 2, 4).reshape(B * n, H, D).to(s["q"].dtype)
    return attend_result(s, out)


def attend_result(s, out):
    return {"out": out, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def plain_sample(s):
    lg = s["logits"].double()          # 64 bits: draws next to a border of the running sums
    R, V = lg.shape
    T = s["temperature"].double()[:, None]
    order = torch.sort(lg, dim=-1, descending=True, stable=True)
    z = (order.values - order.values[:, :1]) / torch.where(T > 0, T, 1.0)
    w = torch.exp(z)
    rank = torch.arange(V, device="cuda")
    k = s["top_k"][:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    before = w.cumsum(-1) - w
    p = s["top_p"].double()[:, None]
    keep = (p >= 1) | (before < p * w.sum(-1, keepdim=True)) | (rank == 0)
    keep &= (w >= s["min_p"].double()[:, None]) | (rank == 0)
    keep &= (T > 0) | (rank == 0)
    w = torch.zeros_like(w).scatter_(1, order.indices, torch.where(keep, w, 0.0))
    run = w.cumsum(-1)
    token = (run > s["u"].double()[:, None] * run[:, -1:]).int().argmax(-1)
    prob = w.gather(1, token[:, None])[:, 0] / run[:, -1]
    return {"tokens": (token + 1).to(torch.int32), "probs": prob.float()}


# ---- the library's calls ------------------------------------------------------------------------

_contexts = {}


def context():
    """One library context on torch's current stream (handle 1: the default stream)."""
    from asicfortranai_b200.quantized import Context
    stream = torch.cuda.current_stream().cuda_stream or 1
    if stream not in _contexts:
        _contexts[stream] = Context(torch.cuda.current_device(), stream=stream)
    return _contexts[stream]


def prepare_own(s):
    """What a serving program keeps besides the arrays: the context, the cache's description, a workspace."""
    s["ctx"] = context()
    if s["op"] == "attend":
        from asicfortranai_b200.quant8 import KV8Cache
        c = s["case"]
        s["cache"] = KV8Cache(s["ctx"], s["k"].data_ptr(), s["v"].data_ptr(), s["k_scale"].data_ptr(),
                              s["v_scale"].data_ptr(), seqs=c["seqs"], kv_heads=c["kv_heads"], head_dim=c["D"],
                              max_seq=c["max_seq"], block=c["block"], code=c["code"])
        need = s["cache"].attention_workspace(c["heads"], c["seqs"] * c["n"], c["n"])
        s["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")


def own_norm(s):
    from asicfortranai_b200 import quant8
    c = s["case"]
    quant8.rms_norm_quant(s["ctx"], s["x"].data_ptr(), s["weight"].data_ptr(), s["codes"].data_ptr(),
                          s["scales"].data_ptr(), c["rows"], c["dim"], dtype=c["dtype"], code=c["code"],
                          group=c["group"], residual=s["residual"].data_ptr(), residual_out=s["h"].data_ptr(), eps=EPS)
    return norm_result(c, s["h"], s["codes"].view(CODE[c["code"]]), s["scales"])


def own_gemm(s):
    from asicfortranai_b200 import quant8
    c = s["case"]
    quant8.fp8_gemm(s["ctx"], s["x"].data_ptr(), s["xs"].data_ptr(), s["w"].data_ptr(), s["ws"].data_ptr(),
                    s["y"].data_ptr(), c["M"], c["N"], c["K"], dtype=c["dtype"], ldx=s["ldx"], ldw=s["ldw"])
    return s["y"]


def own_attend(s):
    c = s["case"]
    B, n = c["seqs"], c["n"]
    s["cache"].append(s["k_new"].data_ptr(), s["v_new"].data_ptr(), s["row_start"].data_ptr(), s["past"].data_ptr(),
                      B * n, n, dtype=c["dtype"])
    s["cache"].attention(s["q"].data_ptr(), s["out"].data_ptr(), c["heads"], s["row_start"].data_ptr(),
                         s["past"].data_ptr(), B * n, n, scale=c["D"] ** -0.5, dtype=c["dtype"],
                         workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel())
    return attend_result(s, s["out"])


def own_sample(s):
    from asicfortranai_b200 import sampling
    c = s["case"]
    sampling.sample_filtered_rows(s["ctx"], s["logits"].data_ptr(), c["rows"], c["V"], s["u"].data_ptr(),
                                  s["tokens"].data_ptr(), temperature=s["temperature"].data_ptr(),
                                  top_k=s["top_k"].data_ptr(), top_p=s["top_p"].data_ptr(),
                                  min_p=s["min_p"].data_ptr(), probs=s["probs"].data_ptr(), dtype=c["dtype"])
    return {"tokens": s["tokens"], "probs": s["probs"]}


def run(s):
    op = s["op"]
    if own:
        return {"norm": own_norm, "gemm": own_gemm, "attend": own_attend, "sample": own_sample}[op](s)
    return {"norm": plain_norm, "gemm": plain_gemm, "attend": plain_attend, "sample": plain_sample}[op](s)


def work(c):
    z = SIZE[c["dtype"]]
    if c["op"] == "norm":
        n = c["rows"] * c["dim"]
        groups = cdiv(c["dim"], c["group"]) if c["group"] else 1
        return {"bytes": 3 * z * n + n + 4 * c["rows"] * groups + 4 * c["dim"], "flops": 8 * n}
    if c["op"] == "gemm":
        M, N, K = c["M"], c["N"], c["K"]
        kb = cdiv(K, 128)
        return {"bytes": M * K + N * K + 4 * kb * (M + cdiv(N, 128)) + z * M * N, "flops": 2 * M * N * K}
    if c["op"] == "attend":
        n, H, G, D, T = (c[k] for k in ("n", "heads", "kv_heads", "D", "block"))
        past = past_lengths(c)
        keys = sum(p + n for p in past)
        pairs = sum(n * p + n * (n + 1) // 2 for p in past)
        rows = c["seqs"] * n
        scales = sum(cdiv(p + n, T) for p in past)
        # codes and scales read once, new keys and values read and written, queries read, outputs written
        return {"bytes": 2 * G * D * keys + 8 * G * scales + 2 * rows * G * D * (z + 1) + 2 * z * rows * H * D,
                "flops": 4 * H * D * pairs}
    return {"bytes": c["rows"] * (z * c["V"] + 28), "flops": 20 * c["rows"] * c["V"]}


# ---- 64 bits ------------------------------------------------------------------------------------

def exact_codes(v, code):
    """Real values to the nearest code (ties to even), as the numbers the codes are."""
    if code == "int8":
        return v.round().clamp(-127, 127)
    a = v.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)    # e4m3: 3 mantissa bits, least exponent -6
    return torch.copysign((a / step).round() * step, v)


def exact_norm(s):
    c = s["case"]
    h = s["x"].double() + s["residual"].double()
    y = s["weight"].double() * h / ((h ** 2).sum(1, keepdim=True) / c["dim"] + EPS).sqrt()
    group = c["group"] or c["dim"]
    codes, scales = torch.empty_like(y), []
    for a in range(0, c["dim"], group):
        part = y[:, a:a + group]
        m = part.abs().max(1, keepdim=True).values / QMAX[c["code"]]
        codes[:, a:a + group] = exact_codes(part / m.clamp_min(1e-300), c["code"]) * (m if c["code"] == "int8" else 1.0)
        scales.append(m)
    return {"h": h, "codes": codes, "scales": torch.cat(scales, 1)}


def exact_gemm(s):
    c = s["case"]
    M, N, K = c["M"], c["N"], c["K"]
    y = torch.zeros(M, N, dtype=torch.float64, device="cuda")
    column = torch.arange(N, device="cuda") // 128
    for b in range(cdiv(K, 128)):
        k = slice(b * 128, min(K, b * 128 + 128))
        part = s["x"][:, k].view(torch.float8_e4m3fn).double() @ s["w"][:, k].view(torch.float8_e4m3fn).double().t()
        y += part * s["xs"][:, b].double()[:, None] * s["ws"][column, b].double()[None]
    return y


def exact_attend(s):
    c = s["case"]
    B, n, H, G, D, T = (c[k] for k in ("seqs", "n", "heads", "kv_heads", "D", "block"))
    out = torch.empty(B * n, H, D, dtype=torch.float64, device="cuda")
    for b, p0 in enumerate(s["past_host"]):
        values = []
        for name in ("k", "v"):
            codes, scale = s[name][b].double(), s[name + "_scale"][b].double()
            values.append(torch.zeros(G, p0 + n, D, dtype=torch.float64, device="cuda"))
            new = s[name + "_new"][b * n:(b + 1) * n].double().transpose(0, 1)
            done = p0 // T * T
            values[-1][:, :done] = codes[:, :done] * scale[:, : p0 // T].repeat_interleave(T, 1)[..., None]
            for a in range(done, p0 + n, T):
                held, upto = max(0, p0 - a), min(a + T, p0 + n)
                fresh = new[:, max(a, p0) - p0:upto - p0]
                was = scale[:, a // T] if held else torch.zeros_like(scale[:, 0])
                # a scale is kept, and a quotient rounded to a code, as the nearest 32-bit value
                now = torch.maximum(was, (fresh.abs().amax((1, 2)) / QMAX[c["code"]]).float().double())[:, None, None]
                if held:
                    older = codes[:, a:a + held] * was[:, None, None]
                    again = (older.float().double() / now).float().double()
                    values[-1][:, a:a + held] = torch.where(now > was[:, None, None], exact_codes(again, c["code"]) * now, older)
                values[-1][:, max(a, p0):upto] = exact_codes((fresh / now).float().double(), c["code"]) * now
        k, v = values
        at = torch.arange(p0 + n, device="cuda")
        allowed = at[None] <= p0 + torch.arange(n, device="cuda")[:, None]
        for h in range(H):
            score = (s["q"][b * n:(b + 1) * n, h].double() @ k[h * G // H].t()) / math.sqrt(D)
            out[b * n:(b + 1) * n, h] = torch.softmax(score.masked_fill(~allowed, -torch.inf), -1) @ v[h * G // H]
    return {"out": out, "k": None, "v": None, "k_scale": None, "v_scale": None}


def exact_sample(s):
    probs = []
    for r in range(s["case"]["rows"]):
        lg = s["logits"][r].double()
        T, k, p, m, u = (s[f][r].item() for f in ("temperature", "top_k", "top_p", "min_p", "u"))
        if T == 0:
            probs.append(torch.ones_like(lg[0]))
            continue
        ids = torch.sort(lg, descending=True, stable=True).indices
        ids = ids[:k] if k > 0 else ids
        prob = torch.softmax(lg[ids] / T, 0)
        if p < 1:
            ids = ids[: int((prob.cumsum(0) < p).sum()) + 1]
        prob = torch.softmax(lg[ids] / T, 0)
        ids = ids[prob >= m * prob[0]].sort().values
        prob = torch.softmax(lg[ids] / T, 0)
        probs.append(prob[int((prob.cumsum(0) <= u).sum().clamp(max=len(ids) - 1))])
    return {"tokens": None, "probs": torch.stack(probs)}


def exact(c, seed):
    s = prepare(c, seed)
    return {"norm": exact_norm, "gemm": exact_gemm, "attend": exact_attend, "sample": exact_sample}[c["op"]](s)
