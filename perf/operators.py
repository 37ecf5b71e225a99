"""Operators of 8-bit block-scaled models as cases that can be timed and checked: routing limited to groups of experts, weights to e4m3
with a scale per 128 x 128 block, the dense product with bf16 activations quantised on the way, and a layer of routed experts.

Shapes are the repository's own configurations: "qwen" (hidden 2048, 512 experts top-10, intermediate 512, softmax router), "glm" (hidden
4096, 160 experts top-8, intermediate 1536, sigmoid router with a bias), "deepseek" (hidden 7168, 256 experts top-8, intermediate 2048; one
GPU of eight holds 32 of them) and the dense 5120 x 17408 FFN.  Activations are bf16 N(0, 1), router logits N(0, 1), weights N(0, 0.02).

`run` computes the plain form in 32 bits (64 for the router's selection); with `own` it makes the library's calls.
"""
import math

import numpy as np
import torch

own = False

B = 128                    # values a scale covers, along both dimensions of a weight
MODELS = {
    "qwen": dict(H=2048, I=512, E=512, held=512, k=10, groups=1, keep=1, group_top=1, score="softmax", bias=False, renorm=True, scale=1.0),
    "glm": dict(H=4096, I=1536, E=160, held=160, k=8, groups=1, keep=1, group_top=1, score="sigmoid", bias=True, renorm=True, scale=2.5),
    "deepseek": dict(H=7168, I=2048, E=256, held=32, k=8, groups=8, keep=4, group_top=2, score="sigmoid", bias=True, renorm=True, scale=2.5),
}


def listed():
    return [
        # the router of one decoded token: latency
        dict(name="route_b1", op="route", M=1, E=256, k=8, groups=8, keep=4, group_top=2, score="sigmoid", bias=True, renorm=True, scale=2.5),
        # an odd serving batch, softmax scores, the best expert stands for its group, weights as they are
        dict(name="route_softmax_b61", op="route", M=61, E=160, k=6, groups=8, keep=3, group_top=1, score="softmax", bias=False, renorm=False, scale=16.0),
        # the router of a prompt chunk
        dict(name="route_8192", op="route", M=8192, E=256, k=8, groups=8, keep=4, group_top=2, score="sigmoid", bias=True, renorm=True, scale=2.5),
        # a checkpoint being loaded: one big fp32 matrix, and a bf16 one whose sizes are no multiples of a block
        dict(name="quantize_17408x5120", op="quantize", N=17408, K=5120, source="fp32"),
        dict(name="quantize_bf16_2111x1552", op="quantize", N=2111, K=1552, source="bf16"),
        # the dense FFN's down projection of one decoded token
        dict(name="linear_m1", op="linear", M=1, N=5120, K=17408),
        # its gate projection for an odd serving batch
        dict(name="linear_m13", op="linear", M=13, N=17408, K=5120),
        # a short prompt, an odd output width
        dict(name="linear_m333", op="linear", M=333, N=4100, K=7168),
        # a prompt chunk
        dict(name="linear_m4096", op="linear", M=4096, N=17408, K=5120),
        # a layer's routed experts: one decoded token
        dict(name="experts_glm_b1", op="experts", model="glm", M=1),
        # a serving batch over many small experts
        dict(name="experts_qwen_b16", op="experts", model="qwen", M=16),
        # a prompt chunk on one GPU of an expert-parallel layer
        dict(name="experts_deepseek_8192", op="experts", model="deepseek", M=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route", "quantize", "linear", "linear", "linear", "experts", "experts", "experts"])
    if op == "route":
        groups = rng.choice([1, 4, 8])
        E = groups * rng.randint(16, 64)
        sigmoid = rng.random() < 0.6
        return dict(op=op, M=_log(rng, 1, 8192), E=E, k=rng.randint(2, 10), groups=groups, keep=rng.randint(1, groups), group_top=rng.choice([1, 2]),
                    score="sigmoid" if sigmoid else "softmax", bias=rng.random() < 0.6, renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5, 16.0]))
    if op == "quantize":
        return dict(op=op, N=_log(rng, 300, 17000), K=16 * rng.randint(20, 320), source=rng.choice(["fp32", "bf16"]))
    if op == "linear":
        N, K = rng.choice([(17408, 5120), (5120, 17408), (2048, 7168), (7168, 2048), (1000 + rng.randint(0, 4000), 16 * rng.randint(60, 460))])
        return dict(op=op, M=_log(rng, 1, 4000), N=N, K=K)
    model = rng.choice(["qwen", "qwen", "glm", "deepseek"])
    return dict(op=op, model=model, M=_log(rng, 1, 8000 if model == "deepseek" else 2000))


# ---------------------------------------------------------------------------------------------------- inputs
def _up(n, m=B):
    return -(-n // m)


def _router_of(case):
    return MODELS[case["model"]] if case["op"] == "experts" else case


def _weights(g, N, K):
    """Codes and scales as the quantiser leaves them for N(0, 0.02) weights."""
    q = torch.randn(N, K, device="cuda", generator=g, dtype=torch.bfloat16).mul_(100.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    s = (torch.rand(_up(N), _up(K), device="cuda", generator=g) * 0.5 + 0.75) * (0.02 / 100.0)
    return q, s


def _layout(H, I):
    """Byte offsets in an expert's record: codes of gate [I, H], up [I, H], down [H, I], then their fp32 scales, to a multiple of 4096."""
    w, sc = H * I, (H // B) * (I // B) * 4
    return dict(w1=0, w3=w, w2=2 * w, s1=3 * w, s3=3 * w + sc, s2=3 * w + 2 * sc, total=-(-(3 * w + 3 * sc) // 4096) * 4096)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = dict(case=case)
    op = case["op"]
    if op in ("route", "experts"):
        r = _router_of(case)
        st["logits"] = torch.randn(case["M"], r["E"], device="cuda", generator=g)
        st["bias"] = torch.randn(r["E"], device="cuda", generator=g) * 0.1 if r["bias"] else None
    if op == "quantize":
        st["w"] = torch.randn(case["N"], case["K"], device="cuda", generator=g) * 0.02
        if case["source"] == "bf16":
            st["w"] = st["w"].to(torch.bfloat16)
    if op == "linear":
        st["q"], st["s"] = _weights(g, case["N"], case["K"])
        st["x"] = torch.randn(case["M"], case["K"], device="cuda", generator=g).to(torch.bfloat16)
    if op == "experts":
        m = MODELS[case["model"]]
        H, I, L = m["H"], m["I"], _layout(m["H"], m["I"])
        recs = torch.zeros(m["held"], L["total"], dtype=torch.uint8, device="cuda")
        for e in range(m["held"]):
            for w, s, (N, K) in (("w1", "s1", (I, H)), ("w3", "s3", (I, H)), ("w2", "s2", (H, I))):
                q, sc = _weights(g, N, K)
                recs[e, L[w]:L[w] + N * K] = q.view(torch.uint8).view(-1)
                recs[e, L[s]:L[s] + sc.numel() * 4] = sc.view(-1).view(torch.uint8)
        table = torch.zeros(m["E"], dtype=torch.int64, device="cuda")               # 0: held by another GPU
        table[: m["held"]] = recs.data_ptr() + torch.arange(m["held"], device="cuda") * L["total"]
        st["recs"], st["table"] = recs, table
        st["x"] = torch.randn(case["M"], H, device="cuda", generator=g).to(torch.bfloat16)
        st["shared"] = (torch.randn(case["M"], H, device="cuda", generator=g) * 0.1).to(torch.bfloat16)
    return st


# ---------------------------------------------------------------------------------------------------- plain forms
def _route(logits, bias, r):
    """Scores and selection in 64 bits: two experts' scores may be next to each other."""
    M, E = logits.shape
    l = logits.double()
    s = torch.sigmoid(l) if r["score"] == "sigmoid" else torch.exp(l - l.amax(1, keepdim=True))
    if r["score"] == "softmax":
        s = s / s.sum(1, keepdim=True)
    c = s if bias is None else s + bias.double()
    if r["keep"] < r["groups"]:
        by = c.view(M, r["groups"], E // r["groups"])
        value = by.sort(dim=2, descending=True).values[:, :, : r["group_top"]].sum(2)
        best = value.sort(dim=1, descending=True, stable=True).indices[:, : r["keep"]]
        on = torch.zeros(M, r["groups"], dtype=torch.bool, device=c.device).scatter_(1, best, True)
        c = torch.where(on.repeat_interleave(E // r["groups"], 1), c, -math.inf)
    ids = c.sort(dim=1, descending=True, stable=True).indices[:, : r["k"]]
    w = s.gather(1, ids)
    if r["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return ids.to(torch.int32), (w * r["scale"]).float()


def _rows_to_e4m3(x):
    """x [M, K] -> values of the codes and their scales [M, K / 128], both fp32."""
    M, K = x.shape
    v = torch.nn.functional.pad(x.float(), (0, _up(K) * B - K)).view(M, -1, B)
    amax = v.abs().amax(2, keepdim=True)
    q = torch.where(amax > 0, v * 448.0 / amax, 0.0).to(torch.float8_e4m3fn).float()
    return q, amax / 448.0


def _times(x, q, s):
    """Rows [M, K] times the block-scaled matrix [N, K], fp32."""
    (N, K), xq = q.shape, _rows_to_e4m3(x)
    w = q.float() * s.repeat_interleave(B, 0)[:N].repeat_interleave(B, 1)[:, :K]
    return (xq[0] * xq[1]).view(x.shape[0], -1)[:, :K] @ w.T


def _blocks_to_e4m3(w):
    N, K = w.shape
    v = torch.nn.functional.pad(w.float(), (0, _up(K) * B - K, 0, _up(N) * B - N)).view(_up(N), B, _up(K), B)
    amax = v.abs().amax((1, 3), keepdim=True)
    q = torch.where(amax > 0, v * 448.0 / amax, 0.0).to(torch.float8_e4m3fn)
    return q.view(_up(N) * B, -1)[:N, :K].contiguous(), (amax / 448.0).view(_up(N), _up(K))


def _matrix(rec, L, w, s, N, K):
    return rec[L[w]:L[w] + N * K].view(torch.float8_e4m3fn).view(N, K), rec[L[s]:L[s] + (N // B) * (K // B) * 4].view(torch.float32).view(N // B, K // B)


def _experts(st, ids, w):
    m = MODELS[st["case"]["model"]]
    H, I, L = m["H"], m["I"], _layout(m["H"], m["I"])
    x = st["x"]
    part = torch.zeros(x.shape[0], m["k"], H, device=x.device)
    for e in range(m["held"]):
        row, pick = (ids == e).nonzero(as_tuple=True)
        if row.numel():
            rec = st["recs"][e]
            gate, up = (_times(x[row], *_matrix(rec, L, a, b, I, H)) for a, b in (("w1", "s1"), ("w3", "s3")))
            part[row, pick] = _times(gate / (1.0 + torch.exp(-gate)) * up, *_matrix(rec, L, "w2", "s2", H, I))
    return ((part * w[:, :, None]).sum(1) + st["shared"].float()).to(torch.bfloat16)


def run(st):
    case = st["case"]
    op = case["op"]
    r = _router_of(case)
    if own:
        import eke_hive_b200 as E

        if op == "quantize":
            q, s = E.fp8_quantize(st["w"])
            return dict(q=q.view(torch.float8_e4m3fn), s=s)
        if op == "linear":
            xq, xs = E.fp8_quant_rows(st["x"])
            return E.fp8_gemm(E.GMat(E.FMT_FP8_B128, case["N"], case["K"], st["q"], st["s"]), xq, xs)
        ids, w = E.router_grouped_topk(st["logits"], r["k"], r["groups"], r["keep"], group_top=r["group_top"], score=r["score"], bias=st["bias"], renorm=r["renorm"],
                                       scale=r["scale"])
        if op == "route":
            return dict(ids=ids, w=w)
        out = E.moe_fp8(ids, w, st["table"], 0, r["E"], st["x"], r["H"], r["I"], shared=st["shared"])
        return dict(ids=ids, w=w, out=out)
    if op == "quantize":
        q, s = _blocks_to_e4m3(st["w"])
        return dict(q=q, s=s)
    if op == "linear":
        return _times(st["x"], st["q"], st["s"]).to(torch.bfloat16)
    ids, w = _route(st["logits"], st["bias"], r)
    if op == "route":
        return dict(ids=ids, w=w)
    return dict(ids=ids, w=w, out=_experts(st, ids, w))


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "route":
        M, E, k = case["M"], case["E"], case["k"]
        return dict(bytes=4 * M * E + 8 * M * k + (4 * E if case["bias"] else 0), flops=8 * M * E)
    if op == "quantize":
        N, K = case["N"], case["K"]
        return dict(bytes=N * K * (5 if case["source"] == "fp32" else 3) + 4 * _up(N) * _up(K), flops=3 * N * K)
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return dict(bytes=N * K + 4 * _up(N) * _up(K) + 2 * M * K + 2 * M * N, flops=2 * M * N * K)
    m, M = MODELS[case["model"]], case["M"]
    hit = m["held"] * (1.0 - (1.0 - m["k"] / m["E"]) ** M)                          # experts that get a row, on average
    return dict(bytes=hit * _layout(m["H"], m["I"])["total"] + M * (4 * m["E"] + 8 * m["k"] + 6 * m["H"]),
                flops=6.0 * m["H"] * m["I"] * M * m["k"] * m["held"] / m["E"])


# ---------------------------------------------------------------------------------------------------- the definition in 64 bits
def _nearest_e4m3(v):
    """fp64 -> the nearest e4m3 value (even mantissa on a tie), |v| <= 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(v / step) * step


def _exact_rows(x):
    M, K = x.shape
    q, s = torch.zeros(M, K, dtype=torch.float64, device=x.device), []
    for a in range(0, K, B):
        v = x[:, a:a + B].double()
        top = v.abs().max(1).values
        q[:, a:a + B] = torch.where(top[:, None] > 0, _nearest_e4m3(v * 448.0 / top[:, None].clamp_min(1e-300)), 0.0)
        s.append((top / 448.0).float().double())                                    # the scale that is stored
    return q, s


def _exact_times(x, q, s):
    y, (xq, xs) = torch.zeros(x.shape[0], q.shape[0], dtype=torch.float64, device=x.device), _exact_rows(x)
    rows = torch.arange(q.shape[0], device=x.device) // B
    for i, a in enumerate(range(0, q.shape[1], B)):
        y += (xq[:, a:a + B] @ q[:, a:a + B].double().T) * xs[i][:, None] * s[:, i].double()[rows][None, :]
    return y


def _exact_route(logits, bias, r):
    l = logits.cpu().numpy().astype(np.float64)
    s = 1.0 / (1.0 + np.exp(-l)) if r["score"] == "sigmoid" else np.exp(l - l.max(1, keepdims=True))
    if r["score"] == "softmax":
        s /= s.sum(1, keepdims=True)
    c = s + (0.0 if bias is None else bias.cpu().numpy().astype(np.float64))
    M, E = c.shape
    size = E // r["groups"]
    group = np.arange(E) // size
    value = np.sort(c.reshape(M, r["groups"], size), axis=2)[:, :, ::-1][:, :, : r["group_top"]].sum(2)
    rank = np.argsort(np.argsort(-value, axis=1, kind="stable"), axis=1, kind="stable")
    c = np.where(rank[:, group] < r["keep"], c, -np.inf)
    ids = np.argsort(-c, axis=1, kind="stable")[:, : r["k"]]
    w = np.take_along_axis(s, ids, 1)
    if r["renorm"]:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    return torch.from_numpy(ids.astype(np.int32)).to(logits.device), torch.from_numpy(w * r["scale"]).to(logits.device)


def exact(case, seed):
    st = prepare(case, seed)
    op, r = case["op"], _router_of(case)
    if op == "quantize":
        w = st["w"].double()
        N, K = w.shape
        q, s = torch.zeros_like(w), torch.zeros(_up(N), _up(K), dtype=torch.float64, device=w.device)
        for i, a in enumerate(range(0, N, B)):
            v = w[a:a + B]
            top = torch.stack([v[:, b:b + B].abs().max() for b in range(0, K, B)])
            s[i] = top / 448.0
            q[a:a + B] = _nearest_e4m3(v * 448.0 / top.clamp_min(1e-300).repeat_interleave(B)[:K])
        return dict(q=q, s=s)
    if op == "linear":
        return _exact_times(st["x"], st["q"], st["s"])
    ids, w = _exact_route(st["logits"], st["bias"], r)
    if op == "route":
        return dict(ids=ids, w=w)
    H, I, L = r["H"], r["I"], _layout(r["H"], r["I"])
    x, out = st["x"], st["shared"].double()
    for e in torch.unique(ids[ids < r["held"]]).tolist():
        row, pick = (ids == e).nonzero(as_tuple=True)
        rec = st["recs"][e]
        gate = _exact_times(x[row], *_matrix(rec, L, "w1", "s1", I, H))
        y = gate * torch.sigmoid(gate) * _exact_times(x[row], *_matrix(rec, L, "w3", "s3", I, H))
        out.index_add_(0, row, _exact_times(y, *_matrix(rec, L, "w2", "s2", H, I)) * w[row, pick][:, None])
    return dict(ids=ids, w=w, out=out)
