"""Cases and plain forms of the block operators over packed rows.

Three operators that follow one another in a transformer block whose rows are the tokens of
sequences of different lengths laid back to back:

  attention  softmax attention with grouped heads, causal or not, over packed sequences; the
             queries of a sequence are its last rows (all of them for a prompt, one while it
             answers, some for a prompt that is continued)
  linear     out = residual + act(a . w^T + bias)
  norm       x' = x + scale * gate * N_post(y), n = N_pre(x')

``own`` false computes the plain forms in 32 bits; ``own`` true calls the library.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"fp16": 2, "bf16": 5}  # GDC_FLOAT16, GDC_BFLOAT16
ACTS = {"none": 0, "gelu": 1, "relu": 2, "silu": 3}
NORMS = {"none": 0, "layer": 1, "rms": 2}


# ------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one short classification row (32 tokens, 16 heads of 64): latency
        _attention("attention_one_row_l32", "fp16", 16, 16, 64, 1, 32, 32, 32, 1, True, 0),
        # a batch of 32 rows of 64 to 256 tokens with their padding removed, grouped heads
        _attention("attention_batch32_l256", "fp16", 16, 4, 64, 32, 64, 256, 256, 3, True, 1),
        # six prompts of very different lengths in one call, head dimension 128
        _attention("attention_prompts_ragged", "bf16", 32, 8, 128, 6, 100, 3000, 3000, 5, True, 0),
        # one long document
        _attention("attention_prompt_8k", "bf16", 32, 8, 128, 1, 8192, 8192, 8192, 7, True, 0),
        # 48 sequences that answer: one new token each over 500 to 8000 keys
        _attention("attention_answer_48", "fp16", 32, 8, 128, 48, 500, 8000, 1, 9, True, 0),
        # output projection of one token, with its bias and residual (hidden 1024)
        _linear("linear_token", "fp16", 1, 1024, 1024, "none", True, True),
        # an odd number of rows and widths that no tile divides
        _linear("linear_odd", "bf16", 777, 1000, 1336, "silu", False, True),
        # FFN down projection of the packed rows of a batch (4096 -> 1024) with its residual
        _linear("linear_ffn_down", "fp16", 4885, 1024, 4096, "none", True, True),
        # a wide up projection over a large batch
        _linear("linear_large", "bf16", 8192, 8192, 4096, "gelu", True, True),
        # one token between two blocks
        _norm("norm_token", "fp16", 1, 1024, "layer", "layer", "column", 1.0),
        # the packed rows of a batch, one gate row for each sequence
        _norm("norm_batch", "fp16", 4885, 1024, "layer", "layer", "sequence", 0.5),
        # a wide residual stream over a long batch
        _norm("norm_wide", "bf16", 16384, 4096, "rms", "rms", "column", 1.0),
    ]


def _attention(name, dtype, heads, kv_heads, dim, batch, low, high, queries, mix, causal, fused):
    """``batch`` sequences of ``low`` to ``high`` keys (by ``mix``), the last ``queries`` rows of each
    at most being queries; fused: q, k and v are column blocks of one projection output."""
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "batch": batch,
            "low": low, "high": high, "queries": queries, "mix": mix, "causal": causal, "fused": bool(fused)}


def _linear(name, dtype, m, n, k, act, bias, residual):
    return {"name": name, "op": "linear", "dtype": dtype, "m": m, "n": n, "k": k, "act": act, "bias": bias, "residual": residual}


def _norm(name, dtype, rows, cols, post, pre, gate, scale):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "cols": cols, "post": post, "pre": pre, "gate": gate,
            "scale": scale}


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm, odd ones among them."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "linear", "norm"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "linear":
        m, n, k = _spread(rng, 1, 8192), _spread(rng, 64, 8192), 8 * _spread(rng, 8, 512)
        c = _linear("", dtype, m, n, k, rng.choice(list(ACTS)), rng.random() < 0.7, rng.random() < 0.8)
    elif op == "norm":
        rows, cols = _spread(rng, 1, 16384), _spread(rng, 64, 4096)
        if rng.random() < 0.6:
            cols = max(64, cols // 8 * 8)
        kinds = rng.choice([("layer", "layer"), ("rms", "rms"), ("none", "layer"), ("none", "rms"), ("rms", "none")])
        c = _norm("", dtype, rows, cols, *kinds, rng.choice(["none", "column", "sequence", "token"]), rng.choice([1.0, 0.5, 0.1767767]))
    else:
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4])
        batch = _spread(rng, 1, 48)
        form = rng.choice(["prompt", "prompt", "answer", "continue"])
        # a prompt batch holds at most 8192 rows, a batch that answers at most 200,000 keys
        high = _spread(rng, 1, 8192 // batch if form == "prompt" else min(8192, 200000 // batch))
        low = _spread(rng, 1, high)
        queries = {"prompt": high, "answer": 1, "continue": max(1, min(high, 2048 // batch) // rng.choice([1, 3, 9]))}[form]
        c = _attention("", dtype, heads, kv_heads, dim, batch, low, high, queries, rng.randrange(1 << 20), rng.random() < 0.8,
                       form == "prompt" and rng.random() < 0.5)
    del c["name"]
    return c


def _lengths(case):
    """Key and query rows of every sequence: part of the case, the same for every seed."""
    rng = random.Random(case["mix"])
    keys = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
    return keys, [min(n, case["queries"]) for n in keys]


def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


# ------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(t)

    s = {"case": case}
    if case["op"] == "attention":
        keys, queries = _lengths(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        tq, tk = sum(queries), sum(keys)
        if case["fused"]:  # the fused projection's output: q | k | v column blocks
            qkv = normal(tk, (h + 2 * hk) * d)
            s["q"], s["k"], s["v"] = qkv[:, :h * d], qkv[:, h * d:(h + hk) * d], qkv[:, (h + hk) * d:]
        else:
            s["q"], s["k"], s["v"] = normal(tq, h * d), normal(tk, hk * d), normal(tk, hk * d)
        s["q_off"] = torch.tensor(_offsets(queries), dtype=torch.int32, device="cuda")
        s["k_off"] = torch.tensor(_offsets(keys), dtype=torch.int32, device="cuda")
        s["scale"] = 1.0 / math.sqrt(d)
        s["out"] = torch.empty(tq, h * d, dtype=t, device="cuda")
    elif case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["w"] = normal(m, k), normal(n, k, std=1.0 / math.sqrt(k))
        s["bias"] = normal(n, std=0.1) if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
        s["out"] = torch.empty(m, n, dtype=t, device="cuda")
    else:
        rows, cols = case["rows"], case["cols"]
        s["y"], s["x"] = normal(rows, cols, std=2.0), normal(rows, cols, std=3.0)
        for at in ("post", "pre"):
            s[at + "_w"] = normal(cols, std=0.1, mean=1.0) if case[at] != "none" else None
            s[at + "_b"] = normal(cols, std=0.1) if case[at] == "layer" else None
        gates = {"none": 0, "column": 1, "sequence": max(1, rows // 150), "token": rows}[case["gate"]]
        s["gate"] = normal(gates, cols, std=0.5) if gates else None
        s["gate_index"] = None
        if case["gate"] == "sequence":  # the sequence of every packed row
            s["gate_index"] = (torch.arange(rows, device="cuda") * gates // rows).to(torch.int32)
        s["x_out"], s["n_out"] = torch.empty_like(s["x"]), torch.empty_like(s["x"]) if case["pre"] != "none" else None
    return s


# ------------------------------------------------------------------------------------- passes

def run(s):
    op = s["case"]["op"]
    if own:
        return {"attention": _own_attention, "linear": _own_linear, "norm": _own_norm}[op](s)
    return {"attention": _plain_attention, "linear": _plain_linear, "norm": _plain_norm}[op](s)


def _plain_attention(s):
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    tq, tk = s["q"].shape[0], s["k"].shape[0]
    q = s["q"].float().reshape(tq, hk, h // hk, d).permute(1, 2, 0, 3).reshape(hk, h // hk * tq, d)
    k = s["k"].float().reshape(tk, hk, d).transpose(0, 1)
    v = s["v"].float().reshape(tk, hk, d).transpose(0, 1)
    # each row's sequence and its place in it, counted from the sequence's end
    q_at, k_at = torch.arange(tq, device=q.device), torch.arange(tk, device=q.device)
    q_seq = torch.searchsorted(s["q_off"], q_at, right=True) - 1
    k_seq = torch.searchsorted(s["k_off"], k_at, right=True) - 1
    hidden = q_seq[:, None] != k_seq[None, :]
    if c["causal"]:
        hidden |= (q_at - s["q_off"][q_seq + 1])[:, None] < (k_at - s["k_off"][k_seq + 1])[None, :]
    p = torch.matmul(q, k.transpose(1, 2)).mul_(s["scale"]).reshape(hk, h // hk, tq, tk)
    p.masked_fill_(hidden, -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(hk, h // hk * tq, tk), v).reshape(hk, h // hk, tq, d).div_(total)
    return o.permute(2, 0, 1, 3).reshape(tq, h * d).to(s["q"].dtype)


def _plain_linear(s):
    z = torch.matmul(s["a"].float(), s["w"].float().t())
    if s["bias"] is not None:
        z += s["bias"].float()
    act = s["case"]["act"]
    if act == "gelu":
        z = 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    elif act == "relu":
        z = torch.where(z > 0, z, torch.zeros_like(z))
    elif act == "silu":
        z = z / (1.0 + torch.exp(-z))
    if s["residual"] is not None:
        z += s["residual"].float()
    return z.to(s["a"].dtype)


EPS = 1e-6


def _plain_normed(z, kind, w, b):
    if kind == "layer":
        z = z - z.mean(-1, keepdim=True)
    z = z / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS) * w.float()
    return z if b is None else z + b.float()


def _plain_norm(s):
    c = s["case"]
    z = s["y"].float()
    if c["post"] != "none":
        z = _plain_normed(z, c["post"], s["post_w"], s["post_b"])
    if s["gate"] is not None:
        z = z * (s["gate"].float() if s["gate_index"] is None else s["gate"].float()[s["gate_index"].long()])
    x = s["x"].float() + c["scale"] * z
    outs = {"x": x.to(s["x"].dtype)}
    if c["pre"] != "none":
        outs["n"] = _plain_normed(x, c["pre"], s["pre_w"], s["pre_b"]).to(s["x"].dtype)
    return outs


def _lib():
    from gliner_decide_metal_b200._lib import lib
    return lib


def _ok(lib, status):
    if status != 0:
        raise RuntimeError(lib.gdc_last_error().decode())


def _at(t):
    return None if t is None else t.data_ptr()


def _own_attention(s):
    c, lib = s["case"], _lib()
    q, k, v, out, q_off, k_off = s["q"], s["k"], s["v"], s["out"], s["q_off"], s["k_off"]
    if "workspace" not in s:  # kept with the buffers, as a program keeps it
        import ctypes
        size = ctypes.c_size_t()
        _ok(lib, lib.gdc_packed_attention_workspace(c["batch"], q.shape[0], k.shape[0], c["heads"], c["kv_heads"], c["dim"],
                                                    ctypes.byref(size)))
        s["workspace"] = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    ws = s["workspace"]
    _ok(lib, lib.gdc_packed_attention(CODES[c["dtype"]], q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(),
                                      v.stride(0), out.data_ptr(), out.stride(0), q_off.data_ptr(), k_off.data_ptr(), c["batch"],
                                      q.shape[0], k.shape[0], c["heads"], c["kv_heads"], c["dim"], int(c["causal"]), s["scale"],
                                      ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    return out


def _own_linear(s):
    c, lib = s["case"], _lib()
    a, w, r, out = s["a"], s["w"], s["residual"], s["out"]
    _ok(lib, lib.gdc_linear_residual(CODES[c["dtype"]], a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(0), _at(s["bias"]), _at(r),
                                     0 if r is None else r.stride(0), out.data_ptr(), out.stride(0), c["m"], None, c["n"], c["k"],
                                     ACTS[c["act"]], torch.cuda.current_stream().cuda_stream))
    return out


def _own_norm(s):
    c, lib = s["case"], _lib()
    y, x, g, n = s["y"], s["x"], s["gate"], s["n_out"]
    cols = c["cols"]
    _ok(lib, lib.gdc_gated_residual_norm(CODES[c["dtype"]], y.data_ptr(), cols, x.data_ptr(), cols, NORMS[c["post"]], _at(s["post_w"]),
                                         _at(s["post_b"]), _at(g), 0 if g is None else g.shape[0], _at(s["gate_index"]), c["scale"],
                                         NORMS[c["pre"]], _at(s["pre_w"]), _at(s["pre_b"]), s["x_out"].data_ptr(), cols, _at(n), cols,
                                         c["rows"], None, cols, EPS, torch.cuda.current_stream().cuda_stream))
    return {"x": s["x_out"]} if n is None else {"x": s["x_out"], "n": n}


# --------------------------------------------------------------------------------- least work

def work(case):
    if case["op"] == "attention":
        keys, queries = _lengths(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(lq * lk - (lq * (lq - 1) // 2 if case["causal"] else 0) for lq, lk in zip(queries, keys))
        return {"bytes": 2 * d * (2 * sum(queries) * h + 2 * sum(keys) * hk) + 8 * (case["batch"] + 1), "flops": 4 * d * h * pairs}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * (m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)),
                "flops": 2 * m * n * k}
    rows, cols = case["rows"], case["cols"]
    gates = {"none": 0, "column": 1, "sequence": max(1, rows // 150), "token": rows}[case["gate"]]
    each = 3 if case["pre"] == "none" else 4
    return {"bytes": 2 * cols * (rows * each + gates) + 2 * cols * 4 + (4 * rows if case["gate"] == "sequence" else 0),
            "flops": 20 * rows * cols}


# --------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        keys, queries = _lengths(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        q_at, k_at = _offsets(queries), _offsets(keys)
        out = torch.zeros(sum(queries), h * d, dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            lq, lk = queries[b], keys[b]
            see = torch.ones(lq, lk, dtype=torch.bool, device="cuda")
            if case["causal"]:
                see = see.tril(lk - lq)
            for head in range(h):
                kv = head // (h // hk)
                q = s["q"][q_at[b]:q_at[b + 1], head * d:(head + 1) * d].double()
                k = s["k"][k_at[b]:k_at[b + 1], kv * d:(kv + 1) * d].double()
                v = s["v"][k_at[b]:k_at[b + 1], kv * d:(kv + 1) * d].double()
                weight = torch.softmax((q @ k.t() * s["scale"]).masked_fill(~see, -math.inf), -1)
                out[q_at[b]:q_at[b + 1], head * d:(head + 1) * d] = weight @ v
        return out
    if case["op"] == "linear":
        z = s["a"].double() @ s["w"].double().t()
        z = z if s["bias"] is None else z + s["bias"].double()
        z = {"none": lambda u: u, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "silu": torch.nn.functional.silu}[case["act"]](z)
        return z if s["residual"] is None else z + s["residual"].double()

    def normed(z, kind, w, b):
        if kind == "none":
            return z
        mean = z.mean(-1, keepdim=True) if kind == "layer" else 0.0
        z = (z - mean) * torch.rsqrt((z - mean).square().mean(-1, keepdim=True) + EPS)
        return z * w.double() + (0.0 if b is None else b.double())

    z = normed(s["y"].double(), case["post"], s["post_w"], s["post_b"])
    if s["gate"] is not None:
        z = z * (s["gate"].double() if s["gate_index"] is None else s["gate"].double().index_select(0, s["gate_index"].long()))
    x = s["x"].double() + case["scale"] * z
    return {"x": x} if case["pre"] == "none" else {"x": x, "n": normed(x, case["pre"], s["pre_w"], s["pre_b"])}
