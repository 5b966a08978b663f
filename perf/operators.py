"""Cases of the operators of quantised language models: matrix-vector products with 4-bit weights and
group scales, int8 products grouped by expert, and the plan that groups tokens by expert.

All of it is integer arithmetic with one right answer.  With ``own`` false, ``run`` computes it with
elementary torch operations (float64 matrix products are exact here: no sum comes near 2^53); with
``own`` true it calls ``mind_b200.blas``.
"""
import math

import numpy as np
import torch

own = False

# ------------------------------------------------------------------------------- cases
# op "plan":    count = tokens * per ids are grouped into `experts`; `pad` tokens at the end of the batch are padding.
# op "w4":      `tokens` activations of kind i8 / i16 / q16 times one 4-bit matrix of rows x cols.
# op "w4g":     the same for routed tokens: every expert has its own matrix, tokens * per slots in all.
# op "grouped": int8, tokens * per rows (rows gathered from the tokens where `gather`), bt: weights given N x K;
#               scaled: each output is multiplied by its expert's column scale and shifted.


def listed():
    return [
        # one decode step of eight sequences, eight experts a token
        {"name": "plan-decode", "op": "plan", "tokens": 8, "per": 8, "experts": 64, "pad": 0},
        # a prefill batch, eight of 256 experts
        {"name": "plan-prefill", "op": "plan", "tokens": 8192, "per": 8, "experts": 256, "pad": 0},
        # a padded batch of odd length: long documents, six of 160 experts
        {"name": "plan-padded", "op": "plan", "tokens": 50021, "per": 6, "experts": 160, "pad": 1777},
        # the smallest call of a decoder layer: one token through a square projection
        {"name": "w4-q16-one", "op": "w4", "kind": "q16", "tokens": 1, "rows": 4096, "cols": 4096, "group": 128},
        # the largest matrix of a decode step, one token, int8 activations
        {"name": "w4-i8-wide", "op": "w4", "kind": "i8", "tokens": 1, "rows": 28672, "cols": 8192, "group": 128},
        # five sequences (a short speculative draft), odd row count, fine groups
        {"name": "w4-i16-draft", "op": "w4", "kind": "i16", "tokens": 5, "rows": 12289, "cols": 5120, "group": 64},
        # eight sequences in one step, Q16.16 activations, the finest groups
        {"name": "w4-q16-eight", "op": "w4", "kind": "q16", "tokens": 8, "rows": 8192, "cols": 8192, "group": 32},
        # one decode step through experts with 4-bit weights: four of 32 experts a token
        {"name": "w4g-i8-decode", "op": "w4g", "kind": "i8", "tokens": 16, "per": 4, "experts": 32, "rows": 2048,
         "cols": 4096, "group": 128},
        # one decode step through int8 experts: a few rows each, all weights are read
        {"name": "grouped-decode", "op": "grouped", "tokens": 32, "per": 4, "experts": 64, "k": 2048, "n": 2816,
         "bt": False, "gather": True, "scaled": True},
        # a prefill batch through the experts' first product: rows gathered from the tokens, requantised
        {"name": "grouped-prefill", "op": "grouped", "tokens": 8192, "per": 4, "experts": 16, "k": 4096, "n": 4096,
         "bt": False, "gather": True, "scaled": True},
        # the second product of a middling batch: rows already in expert order, weights stored N x K, plain sums
        {"name": "grouped-bt", "op": "grouped", "tokens": 2048, "per": 2, "experts": 8, "k": 4096, "n": 2048,
         "bt": True, "gather": False, "scaled": False},
        # odd sizes throughout: no row pitch is a multiple of 16 bytes
        {"name": "grouped-odd", "op": "grouped", "tokens": 389, "per": 2, "experts": 5, "k": 1001, "n": 1283,
         "bt": False, "gather": True, "scaled": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "w4", "w4", "w4g", "grouped", "grouped", "grouped"])
    if op == "plan":
        tokens = _log_int(rng, 1, 100000)
        experts = _log_int(rng, 4, 512)
        return {"op": op, "tokens": tokens, "per": rng.randint(1, min(8, experts)), "experts": experts,
                "pad": rng.choice([0, tokens // 9])}
    if op in ("w4", "w4g"):
        kind = rng.choice(["i8", "i16", "q16"])
        group = rng.choice([32, 64, 128, 256])
        # a column count is a whole number of 32-weight blocks in nearly every model; one in five is not
        cols = 32 * _log_int(rng, 8, 320) if rng.random() < 0.8 else _log_int(rng, 250, 4000)
        if op == "w4":
            return {"op": op, "kind": kind, "tokens": _log_int(rng, 1, 32), "rows": _log_int(rng, 100, 16384),
                    "cols": cols, "group": group}
        experts = _log_int(rng, 4, 64)
        return {"op": op, "kind": kind, "tokens": _log_int(rng, 1, 64), "per": rng.randint(1, min(6, experts)),
                "experts": experts, "rows": _log_int(rng, 100, 2048), "cols": min(cols, 4096), "group": group}
    experts = _log_int(rng, 2, 96)
    aligned = rng.random() < 0.75
    k = 16 * _log_int(rng, 8, 256) if aligned else _log_int(rng, 100, 2000)
    n = 16 * _log_int(rng, 8, 256) if aligned else _log_int(rng, 100, 2000)
    while experts * k * n > 600_000_000:
        experts //= 2
    return {"op": op, "tokens": _log_int(rng, 1, 8192), "per": rng.randint(1, min(4, experts)), "experts": experts,
            "k": k, "n": n, "bt": rng.random() < 0.4, "gather": rng.random() < 0.6, "scaled": rng.random() < 0.6}


# ------------------------------------------------------------------------------ inputs
SHIFT_W4 = {"i8": 6, "i16": 12, "q16": 20}
SHIFT_GROUPED = 12
ITEM = {"i8": 1, "i16": 2, "q16": 4}
DTYPE = {"i8": torch.int8, "i16": torch.int16, "q16": torch.int32}


def _normal_int(g, shape, std, lo, hi, dtype):
    """Rounded normal values, made in pieces so that large matrices do not need a float copy of themselves."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        m = min(step, flat.numel() - i)
        flat[i:i + m] = torch.randn(m, generator=g, device="cuda").mul_(std).round_().clamp_(lo, hi).to(dtype)
    return out


def _activations(g, kind, shape):
    if kind == "i8":  # quantised to the row's largest value
        return _normal_int(g, shape, 34.0, -127, 127, torch.int8)
    if kind == "i16":
        return _normal_int(g, shape, 7000.0, -32767, 32767, torch.int16)
    return _normal_int(g, shape, 1.3 * 65536, -(2 ** 31) + 128, 2 ** 31 - 128, torch.int32)


def _packed(g, lead, rows, cols):
    """4-bit weights, rounded normal in [-8, 7], two a byte, the even column in the low half."""
    pitch = (cols + 1) // 2
    lo = _normal_int(g, (*lead, rows, pitch), 2.3, -8, 7, torch.int8)
    hi = _normal_int(g, (*lead, rows, pitch), 2.3, -8, 7, torch.int8)
    return (lo & 15) | (hi << 4)


def _chosen(g, tokens, per, experts):
    """The experts of every token: distinct, some experts far more popular than others."""
    popular = torch.randn(experts, generator=g, device="cuda").mul_(1.2)
    u = torch.rand((tokens, experts), generator=g, device="cuda").clamp_(1e-6, 1 - 1e-6)
    return (popular - torch.log(-torch.log(u))).topk(per, dim=1).indices.to(torch.int32).contiguous()


def _grouped_by_expert(ids, experts, per):
    key = torch.where((ids >= 0) & (ids < experts), ids, experts).to(torch.int64)
    order = torch.sort(key, stable=True).indices
    counts = torch.zeros(experts + 1, dtype=torch.int64, device="cuda").index_add_(0, key, torch.ones_like(key))
    ends = counts[:experts].cumsum(0)
    offsets = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    return offsets, (order // per).to(torch.int32), order


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    op = case["op"]
    if op == "plan":
        ids = _chosen(g, case["tokens"], case["per"], case["experts"])
        if case["pad"]:
            ids[case["tokens"] - case["pad"]:] = -1
        count = ids.numel()
        s.update(ids=ids.view(-1), count=count,
                 offsets=torch.zeros(case["experts"] + 1, dtype=torch.int32, device="cuda"),
                 # what lies behind the last grouped row is not written
                 order=torch.zeros(count, dtype=torch.int32, device="cuda"),
                 place=torch.zeros(count, dtype=torch.int32, device="cuda"))
        return s
    if op == "grouped":
        m = case["tokens"] * case["per"]
        ids = _chosen(g, case["tokens"], case["per"], case["experts"]).view(-1)
        offsets, rows, _ = _grouped_by_expert(ids, case["experts"], case["per"])
        k, n, e = case["k"], case["n"], case["experts"]
        s.update(m=m, offsets=offsets, ends=offsets.tolist(), rows=rows if case["gather"] else None,
                 a=_activations(g, "i8", (case["tokens"] if case["gather"] else m, k)),
                 b=_normal_int(g, (e, n, k) if case["bt"] else (e, k, n), 30.0, -127, 127, torch.int8),
                 scale=(torch.rand((e, n), generator=g, device="cuda") * 900 + 100).to(torch.int32)
                 if case["scaled"] else None,
                 c=torch.zeros((m, n), dtype=torch.int32, device="cuda"))
        return s
    lead = (case["experts"],) if op == "w4g" else ()
    groups = -(-case["cols"] // case["group"])
    s.update(w=_packed(g, lead, case["rows"], case["cols"]),
             scale=(torch.rand((*lead, case["rows"], groups), generator=g, device="cuda") * 6000 + 500).to(torch.int16),
             x=_activations(g, case["kind"], (case["tokens"], case["cols"])))
    slots = case["tokens"]
    if op == "w4g":
        slots *= case["per"]
        ids = _chosen(g, case["tokens"], case["per"], case["experts"]).view(-1)
        offsets, rows, _ = _grouped_by_expert(ids, case["experts"], case["per"])
        s.update(offsets=offsets, ends=offsets.tolist(), rows_of=rows)
    s["y"] = torch.zeros((slots, case["rows"]), dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------------- plain forms
def _wrap32(v):
    """The low 32 bits of int64 values, as int32."""
    return ((v + 2 ** 31) % 2 ** 32 - 2 ** 31).to(torch.int32)


def _plain_w4(w, scale, x, cols, group, shift):
    """x[t, k] against one packed matrix: the sums of each group, times its scale, added, shifted."""
    rows, groups = w.shape[0], scale.shape[-1]
    xp = torch.zeros((x.shape[0], groups * group), dtype=torch.float64, device="cuda")
    xp[:, :cols] = x
    xg = xp.view(-1, groups, group).permute(1, 2, 0)
    out = torch.empty((x.shape[0], rows), dtype=torch.int32, device="cuda")
    step = max(1, (1 << 27) // max(1, groups * group))
    for r in range(0, rows, step):
        piece = w[r:r + step]
        half = torch.stack([(piece << 4) >> 4, piece >> 4], dim=-1).view(piece.shape[0], -1)[:, :cols]
        wp = torch.zeros((piece.shape[0], groups * group), dtype=torch.float64, device="cuda")
        wp[:, :cols] = half
        d = torch.matmul(wp.view(-1, groups, group).transpose(0, 1), xg)  # [groups, rows, tokens], exact
        total = (d.to(torch.int64) * scale[r:r + step].t().to(torch.int64)[:, :, None]).sum(0)
        out[:, r:r + step] = _wrap32(total >> shift).t()
    return out


def _plain(s):
    op = s["op"]
    if op == "plan":
        offsets, order, perm = _grouped_by_expert(s["ids"], s["experts"], s["per"])
        kept = torch.arange(s["count"], device="cuda", dtype=torch.int32) < offsets[-1]
        place = torch.empty_like(s["place"])
        place[perm] = torch.where(kept, torch.arange(s["count"], device="cuda", dtype=torch.int32), -1)
        return {"offsets": offsets, "rows": torch.where(kept, order, 0), "place": place}
    if op == "w4":
        return _plain_w4(s["w"], s["scale"], s["x"], s["cols"], s["group"], SHIFT_W4[s["kind"]])
    ends = s["ends"]
    if op == "w4g":
        y = torch.zeros_like(s["y"])
        for e in range(s["experts"]):
            lo, hi = ends[e], ends[e + 1]
            if hi > lo:
                y[lo:hi] = _plain_w4(s["w"][e], s["scale"][e], s["x"][s["rows_of"][lo:hi].long()], s["cols"], s["group"],
                                     SHIFT_W4[s["kind"]])
        return y
    c = torch.zeros_like(s["c"])
    for e in range(s["experts"]):
        lo, hi = ends[e], ends[e + 1]
        if hi <= lo:
            continue
        a = s["a"][s["rows"][lo:hi].long()] if s["gather"] else s["a"][lo:hi]
        b = s["b"][e].double()
        acc = torch.matmul(a.double(), b.t() if s["bt"] else b).to(torch.int64)
        if s["scaled"]:
            acc = (acc * s["scale"][e].to(torch.int64)) >> SHIFT_GROUPED
        c[lo:hi] = _wrap32(acc)
    return c


def run(state):
    if not own:
        return _plain(state)
    from mind_b200 import blas
    s = state
    op = s["op"]
    if op == "plan":
        blas.expert_plan(s["ids"], s["offsets"], s["order"], s["place"], s["count"], s["experts"], s["per"])
        return {"offsets": s["offsets"], "rows": s["order"], "place": s["place"]}
    if op == "w4":
        call = {"i8": blas.gemv_w4_i8, "i16": blas.gemv_w4_i16, "q16": blas.gemv_w4_q16}[s["kind"]]
        call(s["w"], s["scale"], s["x"], s["y"], s["tokens"], s["rows"], s["cols"], s["group"], SHIFT_W4[s["kind"]])
        return s["y"]
    if op == "w4g":
        call = {"i8": blas.gemv_w4_grouped_i8, "i16": blas.gemv_w4_grouped_i16,
                "q16": blas.gemv_w4_grouped_q16}[s["kind"]]
        call(s["w"], s["scale"], s["x"], s["rows_of"], s["offsets"], s["y"], s["tokens"] * s["per"], s["rows"], s["cols"],
             s["group"], SHIFT_W4[s["kind"]], s["experts"], s["tokens"])
        return s["y"]
    call = blas.matmul_grouped_i8_bt if s["bt"] else blas.matmul_grouped_i8
    call(s["a"], s["rows"] if s["gather"] else 0, s["b"], s["offsets"], s["scale"] if s["scaled"] else 0, s["c"],
         s["m"], s["k"], s["n"], s["experts"], s["tokens"] if s["gather"] else s["m"], SHIFT_GROUPED)
    return s["c"]


# ---------------------------------------------------------------------- work and truth
def _used(case):
    """Experts that get a token, counted as if every choice were equally likely (an upper estimate)."""
    miss = (1 - case["per"] / case["experts"]) ** case["tokens"]
    return case["experts"] * (1 - miss)


def work(case):
    op = case["op"]
    if op == "plan":
        count = case["tokens"] * case["per"]
        return {"bytes": 12 * count + 4 * (case["experts"] + 1), "flops": 0}
    if op == "grouped":
        m, k, n = case["tokens"] * case["per"], case["k"], case["n"]
        a = (case["tokens"] if case["gather"] else m) * k + (4 * m if case["gather"] else 0)
        weights = _used(case) * (k * n + (4 * n if case["scaled"] else 0))
        return {"bytes": int(a + weights + 4 * m * n), "flops": 2 * m * k * n}
    slots = case["tokens"] * case.get("per", 1)
    matrices = _used(case) if op == "w4g" else 1
    one = case["rows"] * ((case["cols"] + 1) // 2 + 2 * -(-case["cols"] // case["group"]))
    return {"bytes": int(matrices * one + case["tokens"] * case["cols"] * ITEM[case["kind"]] + 4 * slots * case["rows"]),
            "flops": 2 * slots * case["rows"] * case["cols"]}


def _np_low32(v):
    return (v & 0xFFFFFFFF).astype(np.uint32).view(np.int32)


def _np_w4(w, scale, x, group, shift):
    """One packed matrix against x[t, k], in int64, group by group."""
    t, cols = x.shape
    x = x.astype(np.int64)
    total = np.zeros((t, w.shape[0]), dtype=np.int64)
    for g in range(scale.shape[1]):
        k0, k1 = g * group, min(cols, (g + 1) * group)
        byte = w[:, k0 // 2:(k1 + 1) // 2].astype(np.int16)
        digit = np.empty((w.shape[0], 2 * byte.shape[1]), dtype=np.int64)
        digit[:, 0::2] = ((byte & 15) ^ 8) - 8
        digit[:, 1::2] = (((byte >> 4) & 15) ^ 8) - 8
        digit = digit[:, :k1 - k0]
        for i in range(t):
            total[i] += scale[:, g].astype(np.int64) * (digit @ x[i, k0:k1])
    return _np_low32(total >> shift)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        ids = s["ids"].cpu().numpy()
        kept = np.flatnonzero((ids >= 0) & (ids < case["experts"]))
        order = kept[np.argsort(ids[kept], kind="stable")]
        rows, place = np.zeros(ids.size, np.int32), np.full(ids.size, -1, np.int32)
        rows[:order.size] = order // case["per"]
        place[order] = np.arange(order.size)
        offsets = np.searchsorted(ids[order], np.arange(case["experts"] + 1)).astype(np.int32)
        return {"offsets": offsets, "rows": rows, "place": place}
    slots = case["tokens"] * case.get("per", 1)
    if op in ("w4", "w4g"):
        if slots * case["rows"] * case["cols"] > 1.5e9:
            return None
        w, scale, x = (s[v].cpu().numpy() for v in ("w", "scale", "x"))
        if op == "w4":
            return _np_w4(w, scale, x, case["group"], SHIFT_W4[case["kind"]])
        y = np.zeros((slots, case["rows"]), np.int32)
        rows, ends = s["rows_of"].cpu().numpy(), s["ends"]
        for e in range(case["experts"]):
            if ends[e + 1] > ends[e]:
                y[ends[e]:ends[e + 1]] = _np_w4(w[e], scale[e], x[rows[ends[e]:ends[e + 1]]], case["group"],
                                                SHIFT_W4[case["kind"]])
        return y
    if slots * case["k"] * case["n"] > 1.5e11:
        return None
    # float64 products of int8 values add up exactly (no sum passes 2^53)
    a, b = s["a"].cpu().numpy(), s["b"].cpu().numpy()
    rows = s["rows"].cpu().numpy() if case["gather"] else np.arange(slots)
    c, ends = np.zeros((slots, case["n"]), np.int32), s["ends"]
    for e in range(case["experts"]):
        lo, hi = ends[e], ends[e + 1]
        if hi <= lo:
            continue
        be = b[e].astype(np.float64)
        acc = np.dot(a[rows[lo:hi]].astype(np.float64), be.T if case["bt"] else be).astype(np.int64)
        acc = _np_low32(acc).astype(np.int64)
        if case["scaled"]:
            acc = (acc * s["scale"][e].cpu().numpy().astype(np.int64)) >> SHIFT_GROUPED
        c[lo:hi] = _np_low32(acc)
    return c
