"""Operators that train and serve a model on the library's quantized layers, as a user's program runs them.

Five of them, in two groups that share the sort of rows by group (``moe.compute_permutation``, ``lora.plan``):

  lora_apply      low-rank adapters of many requests beside a shared projection (``lora.apply``)
  lora_backward   its gradient: the input's, added to the frozen projection's, and both factors' (``lora.backward``)
  combine_grad    gradient of ``moe.unpermute``: the expert outputs' and the routing weights' (``moe.unpermute_backward``)
  dispatch_grad   gradient of ``moe.permute``: a token's rows are added up (``moe.permute_backward``)
  gate_grad       gradient of ``moe.gate_softmax_topk`` (``moe.gate_softmax_topk_backward``)

A case is a dict of plain values; ``prepare`` makes what a program holds before the call (activations, adapters, and the
plan of the step: rows sorted by adapter or expert, which all layers of a step share), ``run`` is one pass.

Formulas. Row t has adapter a(t), or none; s, A [r, K], B [N, r] are the adapter's scale and factors:
  lora_apply      h_t = A x_t,  out_t = base_t + s B h_t;  out_t = base_t without an adapter
  lora_backward   g_t = s B^T dout_t,  dx_t = dx_base_t + A^T g_t,  dA = sum_t g_t x_t^T,  dB = s sum_t dout_t h_t^T
  combine_grad    row r of pair (t, k): d_permuted_r = w_tk dout_t,  dw_tk = <dout_t, permuted_r>; zero where a pair is dropped
  dispatch_grad   d_input_t = sum_k d_permuted[row of (t, k)]
  gate_grad       s = sum_k w_k dw_k;  renormalised: dl_e = w_k (dw_k - s) at the chosen e, else 0;
                  not renormalised: dl_e = -p_e s, and + w_k dw_k at the chosen e, p = softmax(l)
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One decoding stream with an adapter on an attention projection: the smallest call.
        {"name": "apply_m1_r16_4096x4096", "kind": "lora_apply", "tokens": 1, "adapters": 8, "active": 8, "without": 0.0,
         "rank": 16, "k": 4096, "n": 4096, "dtype": "bf16"},
        # 48 decoding streams of many users, nearly each with an adapter of its own, on the up projection of an MLP.
        {"name": "apply_m48_r16_4096x14336", "kind": "lora_apply", "tokens": 48, "adapters": 64, "active": 64, "without": 0.1,
         "rank": 16, "k": 4096, "n": 14336, "dtype": "f16"},
        # A step that mixes prompt pieces and decoding streams, ranks padded to 64, on a wide model's down projection.
        {"name": "apply_m777_r64_2048x7168", "kind": "lora_apply", "tokens": 777, "adapters": 24, "active": 24, "without": 0.2,
         "rank": 64, "k": 2048, "n": 7168, "dtype": "bf16"},
        # Prompts of a few tenants, or the forward pass of a training step on long sequences.
        {"name": "apply_m16384_r64_4096x4096", "kind": "lora_apply", "tokens": 16384, "adapters": 8, "active": 8, "without": 0.05,
         "rank": 64, "k": 4096, "n": 4096, "dtype": "bf16"},
        # Gradient of a short batch: several small adapters trained at once.
        {"name": "lora_grad_m1001_r8_2048x4096", "kind": "lora_backward", "tokens": 1001, "adapters": 4, "active": 4, "without": 0.0,
         "rank": 8, "k": 2048, "n": 4096, "dtype": "f16"},
        # Gradient of a long batch with one adapter in training beside one that this batch does not use.
        {"name": "lora_grad_m16384_r64_4096x4096", "kind": "lora_backward", "tokens": 16384, "adapters": 2, "active": 1, "without": 0.0,
         "rank": 64, "k": 4096, "n": 4096, "dtype": "bf16"},
        # A routed layer's way back: a small micro-batch, all experts here.
        {"name": "combine_grad_t48_k8_7168", "kind": "combine_grad", "tokens": 48, "top_k": 8, "experts": 64, "hidden": 7168,
         "dropped": 0.0, "dtype": "bf16"},
        # A training batch over 256 experts, an eighth of the pairs dropped (experts elsewhere, or over capacity).
        {"name": "combine_grad_t4096_k8_7168", "kind": "combine_grad", "tokens": 4096, "top_k": 8, "experts": 256, "hidden": 7168,
         "dropped": 0.125, "dtype": "bf16"},
        # Two experts a token, ragged token count.
        {"name": "dispatch_grad_t333_k2_4096", "kind": "dispatch_grad", "tokens": 333, "top_k": 2, "experts": 8, "hidden": 4096,
         "dropped": 0.0, "dtype": "f16"},
        {"name": "dispatch_grad_t4096_k8_7168", "kind": "dispatch_grad", "tokens": 4096, "top_k": 8, "experts": 256, "hidden": 7168,
         "dropped": 0.125, "dtype": "bf16"},
        # The router of a small batch, weights renormalised over the chosen experts.
        {"name": "gate_grad_t512_e64", "kind": "gate_grad", "tokens": 512, "experts": 64, "top_k": 8, "renormalize": True, "dtype": "f32"},
        # The router of a long batch, plain softmax probabilities as weights.
        {"name": "gate_grad_t16384_e256", "kind": "gate_grad", "tokens": 16384, "experts": 256, "top_k": 8, "renormalize": False,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lora_apply", "lora_apply", "lora_backward", "combine_grad", "dispatch_grad", "gate_grad"])
    if kind in ("lora_apply", "lora_backward"):
        # widths are multiples of 8 elements, 16 bytes, as every model's are; ranks from 8 to 128, token counts any
        k, n = 8 * _log(rng, 64, 1024), 8 * _log(rng, 64, 2048)
        most = 16384 * 12288 // (k + 2 * n) if kind == "lora_apply" else 16384 * 12288 // (2 * k + n)
        adapters = _log(rng, 1, 64)
        return {"kind": kind, "tokens": _log(rng, 1 if kind == "lora_apply" else 16, min(most, 16384)), "adapters": adapters,
                "active": rng.randint(1, adapters), "without": rng.choice([0.0, 0.0, 0.1, 0.5]),
                "rank": rng.choice([8, 16, 16, 24, 32, 64]), "k": k, "n": n, "dtype": rng.choice(["bf16", "f16"])}
    if kind == "gate_grad":
        experts = rng.choice([8, 16, 60, 64, 100, 128, 160, 256])
        return {"kind": kind, "tokens": _log(rng, 16, 16384), "experts": experts, "top_k": rng.randint(1, 8),
                "renormalize": rng.random() < 0.5, "dtype": rng.choice(["f32", "bf16", "f16"])}
    top_k, hidden, dtype = rng.randint(1, 8), 8 * _log(rng, 128, 1024), rng.choice(["bf16", "f16", "bf16", "f32"])
    most = 4096 * 8 * 7168 // (top_k * hidden * (2 if dtype == "f32" else 1))
    return {"kind": kind, "tokens": _log(rng, 1, min(most, 16384)), "top_k": top_k, "experts": rng.choice([8, 16, 64, 256]), "hidden": hidden,
            "dropped": rng.choice([0.0, 0.0, 0.125, 0.875]), "dtype": dtype}


def _sorted_rows(group, groups):
    """Rows in group order (stable), those of no group last, and where each group begins."""
    order = torch.sort(torch.where((group < 0) | (group >= groups), groups, group), stable=True).indices
    counts = torch.bincount(group[(group >= 0) & (group < groups)], minlength=groups)
    offsets = torch.zeros(groups + 2, dtype=torch.int64, device=group.device)
    offsets[1:groups + 1] = counts.cumsum(0)
    offsets[groups + 1] = group.numel()
    return order.to(torch.int32), offsets.to(torch.int32)


def _lora_state(case, g, dev):
    t, l, r, k, n = (case[x] for x in ("tokens", "adapters", "rank", "k", "n"))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dt)

    # adapters of requests: prompts take runs of rows, streams one row each
    ids = torch.randint(0, case["active"], (t,), generator=g, device=dev)
    runs = torch.arange(t, device=dev) // 64
    ids = torch.where(runs % 2 == 0, ids[(runs * 64).clamp(max=t - 1)], ids) if t > 64 else ids
    ids = torch.where(torch.rand(t, generator=g, device=dev) < case["without"], -1, ids)
    order, offsets = _sorted_rows(ids, l)
    s = {"case": case, "ids": ids, "sorted_ids": order, "offsets": offsets,
         "x": normal(t, k), "a": normal(l, r, k, std=k ** -0.5), "b": normal(l, n, r, std=0.05),
         "scales": torch.rand(l, generator=g, device=dev) * 1.5 + 0.5}
    # rows by adapter in a padded table [adapters, longest]: row t of the table means "none"
    counts = (offsets[1:l + 1] - offsets[:l]).long()
    longest = max(1, int(counts.max()))
    at = torch.arange(longest, device=dev)
    place = (offsets[:l].long()[:, None] + at).clamp(max=t - 1)
    s["table"] = torch.where(at < counts[:, None], order.long()[place], t)
    if case["kind"] == "lora_apply":
        s["base"] = normal(t, n)
    else:
        s["dout"], s["dx_base"] = normal(t, n, std=0.02), normal(t, k, std=0.02)
        h = torch.zeros(t + 1, r, device=dev)
        xs = torch.cat([s["x"], s["x"].new_zeros(1, k)])
        for e in range(l):   # what the forward pass kept, adapter by adapter
            h[s["table"][e]] = xs[s["table"][e]].float() @ s["a"][e].float().t()
        s["h"] = h[:t].contiguous()
    return s


def _moe_state(case, g, dev):
    t, k, e, hid = case["tokens"], case["top_k"], case["experts"], case["hidden"]
    dt = DTYPES[case["dtype"]]
    logits = torch.randn(t, e, generator=g, device=dev)
    w, idx = torch.topk(torch.softmax(logits, 1), k, dim=1)
    idx = torch.where(torch.rand(t, k, generator=g, device=dev) < case["dropped"], -1, idx)
    order, offsets = _sorted_rows(idx.flatten(), e)
    # pairs without an expert hold -1 at the end, as the permutation writes it
    ids = torch.where(torch.arange(t * k, device=dev) < offsets[e], order, -1).to(torch.int32)
    s = {"case": case, "sorted_ids": ids, "weights": (w / w.sum(1, keepdim=True)).contiguous()}
    if case["kind"] == "combine_grad":
        s["dout"] = (torch.randn(t, hid, generator=g, device=dev) * 0.02).to(dt)
        s["permuted"] = torch.randn(t * k, hid, generator=g, device=dev).to(dt)
    else:
        s["d_permuted"] = (torch.randn(t * k, hid, generator=g, device=dev) * 0.02).to(dt)
    return s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    if case["kind"] in ("lora_apply", "lora_backward"):
        return _lora_state(case, g, dev)
    if case["kind"] in ("combine_grad", "dispatch_grad"):
        return _moe_state(case, g, dev)
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = (torch.randn(t, e, generator=g, device=dev) * 2).to(DTYPES[case["dtype"]])
    w, idx = torch.topk(torch.softmax(logits.float(), 1), k, dim=1)
    if case["renormalize"]:
        w = w / w.sum(1, keepdim=True)
    return {"case": case, "logits": logits, "weights": w.contiguous(), "indices": idx.to(torch.int32).contiguous(),
            "d_weights": torch.randn(t, k, generator=g, device=dev) * 0.02}


# ---- the framework's operators -------------------------------------------------------------------------
def _run_own(s):
    from kernel_set_b200 import lora, moe
    case = s["case"]
    kind = case["kind"]
    if kind == "lora_apply":
        return lora.apply(torch.empty_like(s["base"]), s["base"], s["x"], s["a"], s["b"], s["scales"], s["sorted_ids"], s["offsets"])
    if kind == "lora_backward":
        return lora.backward(torch.empty_like(s["dx_base"]), torch.empty_like(s["a"]), torch.empty_like(s["b"]), s["dx_base"], s["dout"],
                             s["x"], s["h"], s["a"], s["b"], s["scales"], s["sorted_ids"], s["offsets"])
    t, k = case["tokens"], case["top_k"]
    if kind == "combine_grad":
        return moe.unpermute_backward(torch.empty_like(s["permuted"]), torch.empty_like(s["weights"]), s["dout"], s["permuted"],
                                      s["sorted_ids"], s["weights"], t, k, case["hidden"])
    if kind == "dispatch_grad":
        d_input = torch.empty(t, case["hidden"], dtype=s["d_permuted"].dtype, device=s["d_permuted"].device)
        return moe.permute_backward(d_input, s["d_permuted"], s["sorted_ids"], t, k, case["hidden"])
    return moe.gate_softmax_topk_backward(torch.empty_like(s["logits"]), s["d_weights"], s["weights"], s["indices"], s["logits"], t,
                                          case["experts"], k, renormalize=case["renormalize"])


# ---- plain forms ----------------------------------------------------------------------------------------
def _rows(table, m):
    """The rows of `m` that the padded table names, in fp32; a row of zeros for "none"."""
    return torch.cat([m, m.new_zeros(1, m.shape[1])])[table].float()


def _back(table, rows, t, like):
    """Rows of the padded table back in their places (zeros elsewhere)."""
    out = torch.zeros(t + 1, rows.shape[-1], dtype=torch.float32, device=like.device)
    out[table.flatten()] = rows.flatten(0, 1)
    return out[:t]


def run(state):
    s = state
    if own:
        return _run_own(s)
    case = s["case"]
    kind, t = case["kind"], case["tokens"]
    if kind == "lora_apply":
        h = torch.bmm(_rows(s["table"], s["x"]), s["a"].float().transpose(1, 2))
        d = torch.bmm(h, s["b"].float().transpose(1, 2)) * s["scales"][:, None, None]
        return (s["base"].float() + _back(s["table"], d, t, d)).to(s["base"].dtype)
    if kind == "lora_backward":
        dt = s["a"].dtype
        x, dout, h = _rows(s["table"], s["x"]), _rows(s["table"], s["dout"]), _rows(s["table"], s["h"])
        sc = s["scales"][:, None, None]
        g = torch.bmm(dout, s["b"].float()) * sc
        dx = s["dx_base"].float() + _back(s["table"], torch.bmm(g, s["a"].float()), t, g)
        return dx.to(dt), torch.bmm(g.transpose(1, 2), x).to(dt), (torch.bmm(dout.transpose(1, 2), h) * sc).to(dt)
    k = case["top_k"]
    if kind == "gate_grad":
        w, dw, idx = s["weights"], s["d_weights"], s["indices"].long()
        dot = (w * dw).sum(1, keepdim=True)
        if case["renormalize"]:
            d = torch.zeros(t, case["experts"], device=w.device)
            return d.scatter_add_(1, idx, w * (dw - dot)).to(s["logits"].dtype)
        p = torch.exp(s["logits"].float() - s["logits"].float().amax(1, keepdim=True))
        d = -dot * (p / p.sum(1, keepdim=True))
        return d.scatter_add_(1, idx, w * dw).to(s["logits"].dtype)
    ids = s["sorted_ids"].long()
    live = ids >= 0
    pair = ids.clamp(min=0)
    if kind == "combine_grad":
        dout = s["dout"][pair // k].float()
        dp = torch.where(live[:, None], s["weights"].flatten()[pair][:, None] * dout, 0.0)
        dots = torch.where(live, (dout * s["permuted"].float()).sum(1), 0.0)
        dw = torch.zeros(t * k, device=dots.device).index_add_(0, pair, dots)
        return dp.to(s["permuted"].dtype), dw.view(t, k)
    d = torch.zeros(t, case["hidden"], device=ids.device)
    d.index_add_(0, pair // k, torch.where(live[:, None], s["d_permuted"].float(), 0.0))
    return d.to(s["d_permuted"].dtype)


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind, t = case["kind"], case["tokens"]
    if kind in ("lora_apply", "lora_backward"):
        ids = s["ids"]
        if kind == "lora_apply":
            out = s["base"].double()
            for e in range(case["adapters"]):
                rows = (ids == e).nonzero()[:, 0]
                out[rows] += float(s["scales"][e]) * (s["x"][rows].double() @ s["a"][e].double().t() @ s["b"][e].double().t())
            return out
        dx, da, db = s["dx_base"].double(), torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
        for e in range(case["adapters"]):
            rows = (ids == e).nonzero()[:, 0]
            sc, dout = float(s["scales"][e]), s["dout"][rows].double()
            g = sc * (dout @ s["b"][e].double())
            dx[rows] += g @ s["a"][e].double()
            da[e] = g.t() @ s["x"][rows].double()
            db[e] = sc * (dout.t() @ s["h"][rows].double())
        return dx, da, db
    k = case["top_k"]
    if kind == "gate_grad":
        w, dw, idx = s["weights"].double(), s["d_weights"].double(), s["indices"].long()
        chosen = torch.zeros(t, case["experts"], dtype=torch.float64, device=w.device).scatter(1, idx, dw)
        dot = (w * dw).sum(1, keepdim=True)
        if case["renormalize"]:
            full = torch.zeros_like(chosen).scatter(1, idx, w)
            return full * (chosen - dot)
        return torch.zeros_like(chosen).scatter(1, idx, w) * chosen - torch.softmax(s["logits"].double(), 1) * dot
    # where each pair's row lies, -1 for a dropped pair
    where = torch.full((t * k,), -1, dtype=torch.int64, device=s["sorted_ids"].device)
    rows = (s["sorted_ids"] >= 0).nonzero()[:, 0]
    where[s["sorted_ids"][rows].long()] = rows
    where = where.view(t, k)
    if kind == "dispatch_grad":
        d = torch.zeros(t, case["hidden"], dtype=torch.float64, device=where.device)
        for j in range(k):
            has = where[:, j] >= 0
            d[has] += s["d_permuted"][where[has, j]].double()
        return d
    dp = torch.zeros_like(s["permuted"], dtype=torch.float64)
    dw = torch.zeros(t, k, dtype=torch.float64, device=where.device)
    for j in range(k):
        has = where[:, j] >= 0
        dout = s["dout"][has].double()
        dp[where[has, j]] = s["weights"][has, j].double()[:, None] * dout
        dw[has, j] = (dout * s["permuted"][where[has, j]].double()).sum(1)
    return dp, dw


def work(case):
    kind, t = case["kind"], case["tokens"]
    elt = 4 if case["dtype"] == "f32" else 2
    if kind in ("lora_apply", "lora_backward"):
        k, n, r = case["k"], case["n"], case["rank"]
        have = t * (1 - case["without"])                                # rows with an adapter
        used = case["active"] * (1 - (1 - 1 / case["active"]) ** have)  # adapters that some row has, about
        factors = (k + n) * r * elt
        if kind == "lora_apply":
            return {"bytes": have * k * elt + 2 * t * n * elt + used * factors + 4 * t, "flops": 2 * have * r * (k + n)}
        return {"bytes": have * (k + n) * elt + 2 * t * k * elt + have * r * 4 + (used + case["adapters"]) * factors + 4 * t,
                "flops": 4 * have * r * (k + n)}
    k = case["top_k"]
    if kind == "gate_grad":
        e = case["experts"]
        logits = 0 if case["renormalize"] else t * e * elt
        return {"bytes": logits + t * e * elt + t * k * 12, "flops": t * (4 * e + 4 * k)}
    rows, hid = t * k * (1 - case["dropped"]), case["hidden"]
    if kind == "combine_grad":   # dropped rows are written, with zeros
        return {"bytes": t * hid * elt + rows * hid * elt + t * k * hid * elt + t * k * 12, "flops": 3 * rows * hid}
    return {"bytes": rows * hid * elt + t * hid * elt + t * k * 4, "flops": rows * hid}
