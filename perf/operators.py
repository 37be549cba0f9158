"""Routing, the gated delta rule and the verification of drafted tokens, as measurable cases.

Three operators beside the MoE layer, each through the binding a serving program uses:

* ``route``: router logits [T][E] to expert ids and weights [T][K] (sigmoid or softmax scores, a
  correction bias, expert groups, renormalisation), what k3x_hip_moe_forward_routed takes;
* ``delta``: the gated delta rule over ragged sequences with their states: one token a sequence
  (decode), a few (a verification window, committed up to a length that is on the device) or a
  prompt's chunk (prefill);
* ``verify``: drafted tokens against the target's logits or probabilities, from given uniforms.

``run`` computes the plain form where ``own`` is false and calls the framework where it is true.
"""
import os
import sys

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6  # of the L2 norms of queries and keys
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    delta = dict(kind="delta", dtype="bf16", key_heads=32, value_heads=32, key_dim=128,
                 value_dim=128, gate="channel", norm=True, limits=False)
    return [
        # Routing of a decode step: two positions over the K3-shaped layer's experts.
        dict(kind="route", name="route_t2", tokens=2, experts=384, top_k=16, scoring="sigmoid",
             bias=True, groups=1, top_groups=1, group_score="top2", renorm="float", scale=2.5,
             dtype="fp32"),
        # A prefill chunk of the official layer: 896 experts, contributions renormalised in double.
        dict(kind="route", name="route_official_t2048", tokens=2048, experts=896, top_k=16,
             scoring="sigmoid", bias=True, groups=1, top_groups=1, group_score="top2",
             renorm="double", scale=1.0, dtype="fp32"),
        # Group-limited softmax routing over a large batch of prompts, ragged count, bf16 logits.
        dict(kind="route", name="route_groups_t30011", tokens=30011, experts=256, top_k=8,
             scoring="softmax", bias=True, groups=8, top_groups=4, group_score="top2",
             renorm="float", scale=2.5, dtype="bf16"),
        # One user decoding: the state's read and write, latency.
        dict(delta, name="delta_decode_n1", lens="1"),
        # A batch of users decoding, a token each.
        dict(delta, name="delta_decode_n64", lens="1*64"),
        # A verification window of 8 users' drafts, committed up to the accepted counts.
        dict(delta, name="delta_window_n8", lens="16*8", limits=True),
        # One prefill chunk of one prompt.
        dict(delta, name="delta_prefill_t2048", lens="2048"),
        # A batch of ragged prompts, shared key heads and one decay a head.
        dict(delta, name="delta_ragged_t8192", lens="2047,1500,1,1024,977,1333,1310", key_heads=16,
             gate="head"),
        # Greedy verification of one user's draft: argmax of a few rows of bf16 logits.
        dict(kind="verify", name="verify_greedy_n1", sequences=1, drafts=4, vocab=163840,
             form="logits", dtype="bf16", greedy=True, draft_dist=False, temperature=1.0),
        # Sampled verification from logits, odd vocabulary.
        dict(kind="verify", name="verify_logits_n16", sequences=16, drafts=4, vocab=100003,
             form="logits", dtype="fp32", greedy=False, draft_dist=True, temperature=0.8),
        # A large batch whose sampler has the probabilities already.
        dict(kind="verify", name="verify_probs_n64", sequences=64, drafts=7, vocab=131072,
             form="probs", dtype="fp32", greedy=False, draft_dist=True, temperature=1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    u = rng.random()
    if u < 0.3:
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log_int(rng, max(2, 16 // groups), 896 // groups)
        top_groups = rng.randint(1, groups)
        return dict(kind="route", tokens=_log_int(rng, 1, 30000), experts=experts,
                    top_k=rng.randint(1, min(16, experts // groups * top_groups)),
                    scoring=rng.choice(["sigmoid", "softmax"]), bias=rng.random() < 0.7,
                    groups=groups, top_groups=top_groups, group_score=rng.choice(["max", "top2"]),
                    renorm=rng.choice(["float", "double", "none"]), scale=rng.choice([1.0, 2.5]),
                    dtype=rng.choice(["fp32", "bf16"]))
    if u < 0.75:
        v = rng.random()
        key_heads = rng.choice([1, 2, 4, 8, 16, 32])
        ratio = rng.choice([1, 1, 2, 4])
        if key_heads * ratio > 32:
            ratio = 1
        heads = key_heads * ratio
        key_dim, value_dim = rng.choice([(128, 128), (64, 64), (128, 64), (96, 80), (64, 128),
                                         (33, 47)])
        if v < 0.35:  # decode and windows
            n, most = _log_int(rng, 1, 64), rng.choice([1, 1, 5, 16])
            lens = [rng.randint(1 if most == 1 else 0, most) for _ in range(n)]
        else:
            n = rng.randint(1, 6)
            total = _log_int(rng, 32, 8192 * 32 // max(heads, 32))
            lens = [max(1, int(total / n * (0.4 + 1.2 * rng.random()) / 1.6)) for _ in range(n)]
        if not sum(lens):
            lens[0] = 1
        return dict(kind="delta", dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    key_heads=key_heads, value_heads=heads, key_dim=key_dim, value_dim=value_dim,
                    gate=rng.choice(["channel", "head", "none"]), norm=True,
                    limits=rng.random() < 0.3, lens=",".join(map(str, lens)))
    form = rng.choice(["logits", "logits", "probs"])
    return dict(kind="verify", sequences=_log_int(rng, 1, 48), drafts=rng.randint(1, 7),
                vocab=_log_int(rng, 1000, 131072), form=form,
                dtype=rng.choice(["fp32", "bf16"]) if form == "logits" else "fp32",
                greedy=form == "logits" and rng.random() < 0.3, draft_dist=rng.random() < 0.6,
                temperature=rng.choice([1.0, 0.7]) if form == "logits" else 1.0)


def _lens(c):
    out = []
    for part in c["lens"].split(","):
        n, _, times = part.partition("*")
        out += [int(n)] * int(times or 1)
    return out


def work(c):
    if c["kind"] == "route":
        T, E, K = c["tokens"], c["experts"], c["top_k"]
        es = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": T * E * es + (E * 4 if c["bias"] else 0) + T * K * 8,
                "flops": 30 * T * E}
    if c["kind"] == "delta":
        lens = _lens(c)
        T, N = sum(lens), len(lens)
        Hk, H, K, V = c["key_heads"], c["value_heads"], c["key_dim"], c["value_dim"]
        es = 4 if c["dtype"] == "fp32" else 2
        g = {"channel": K, "head": 1, "none": 0}[c["gate"]]
        return {"bytes": 2 * T * Hk * K * es + 2 * T * H * V * es + T * H * (g + 1) * 4
                + 2 * N * H * K * V * 4,
                "flops": 7 * T * H * K * V}
    N, D, V = c["sequences"], c["drafts"], c["vocab"]
    es = 4 if c["dtype"] == "fp32" else 2
    if c["form"] == "probs":  # the drafted tokens' values and the row that is sampled from
        rows = N * (2 if c["draft_dist"] else 1)
    else:
        rows = N * (D + 1 + (D if c["draft_dist"] and not c["greedy"] else 0))
    return {"bytes": rows * V * es + N * (D + 1) * 12, "flops": 20 * rows * V}


# ---- inputs -----------------------------------------------------------------------------------

def _gen(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1_000_003 + stream) % (1 << 62))
    return g


def _normal(seed, stream, *shape):
    return torch.randn(shape, device=DEV, generator=_gen(seed, stream))


def _uniform(seed, stream, *shape):
    return torch.rand(shape, device=DEV, generator=_gen(seed, stream))


def _binding():
    path = os.path.join(os.getcwd(), "project-k3x_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import k3x_amd
    return k3x_amd


_CONTEXT = []


def _context():
    """The program's one context, kept as a server keeps it."""
    if not _CONTEXT:
        _CONTEXT.append(_binding().Context(0))
    return _CONTEXT[0]


def prepare(c, seed):
    s = dict(case=c)
    if c["kind"] == "route":
        T, E, K = c["tokens"], c["experts"], c["top_k"]
        s["logits"] = (_normal(seed, 1, T, E) * 1.7).to(DTYPES[c["dtype"]])
        s["bias"] = _normal(seed, 2, E) * (0.1 if c["scoring"] == "sigmoid" else 0.005) \
            if c["bias"] else None
        s["ids"] = torch.empty((T, K), dtype=torch.int32, device=DEV)
        s["weights"] = torch.empty((T, K), device=DEV)
        return s
    if c["kind"] == "delta":
        lens = _lens(c)
        T, N, most = sum(lens), len(lens), max(lens)
        Hk, H, K, V = c["key_heads"], c["value_heads"], c["key_dim"], c["value_dim"]
        dt = DTYPES[c["dtype"]]
        s["q"], s["k"] = _normal(seed, 1, T, Hk, K).to(dt), _normal(seed, 2, T, Hk, K).to(dt)
        s["v"] = _normal(seed, 3, T, H, V).to(dt)
        s["beta"] = torch.sigmoid(_normal(seed, 4, T, H))
        # Log decays -A softplus(x + b): A in 1..16 a head, softplus(b) in 0.001..0.1.
        s["gate"] = None
        if c["gate"] != "none":
            n = K if c["gate"] == "channel" else 1
            a = 1 + 15 * _uniform(seed, 5, H, 1)
            step = 0.001 * 100 ** _uniform(seed, 6, H, n)
            x = 0.5 * _normal(seed, 7, T, H, n) + torch.log(torch.expm1(step))
            s["gate"] = -a * torch.nn.functional.softplus(x)
            if n == 1:
                s["gate"] = s["gate"].squeeze(-1).contiguous()
        s["state"] = 0.2 * _normal(seed, 8, N, H, K, V)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        s["offsets"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
        s["limits"] = None
        if c["limits"]:
            s["limits"] = torch.randint(0, most + 1, (N,), device=DEV, dtype=torch.int32,
                                        generator=_gen(seed, 9))
        s["longest"] = most
        s["out"] = torch.zeros((T, H, V), dtype=dt, device=DEV)
        s["state_out"] = torch.zeros_like(s["state"])
        return s
    N, D, V = c["sequences"], c["drafts"], c["vocab"]
    target = _normal(seed, 1, N, D + 1, V) * 2.5
    draft = target[:, :D] + _normal(seed, 2, N, D, V) * 0.8
    if c["greedy"] or not c["draft_dist"]:  # the draft's own best guess
        s["tokens"] = draft.argmax(-1).to(torch.int32)
    else:
        noise = -torch.log(-torch.log(_uniform(seed, 3, N, D, V).clamp(1e-12, 1 - 1e-7)))
        s["tokens"] = (draft / c["temperature"] + noise).argmax(-1).to(torch.int32)
    dt = DTYPES[c["dtype"]]
    if c["form"] == "probs":
        target, draft = torch.softmax(target, -1), torch.softmax(draft, -1)
    s["target"] = target.to(dt)
    s["draft"] = draft.to(dt) if c["draft_dist"] and not c["greedy"] else None
    s["accept_u"] = _uniform(seed, 4, N, D)
    s["sample_u"] = _uniform(seed, 5, N)
    s["accepted"] = torch.zeros((N,), dtype=torch.int32, device=DEV)
    s["out_tokens"] = torch.zeros((N, D + 1), dtype=torch.int32, device=DEV)
    return s


# ---- the plain forms --------------------------------------------------------------------------

def _plain_route(c, s):
    """Scores as the layer's router forms them: a rounded exponential, an fp32 sum and quotient."""
    l, E, K = s["logits"].float(), c["experts"], c["top_k"]
    if c["scoring"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-l.double()).float())
    else:  # next to another expert's score every bit counts
        e = torch.exp(l.double() - l.double().amax(-1, keepdim=True))
        score = (e / e.sum(-1, keepdim=True)).float()
    adj = score if s["bias"] is None else score + s["bias"]
    if c["groups"] > 1:
        parts = adj.view(adj.shape[0], c["groups"], E // c["groups"])
        if c["group_score"] == "max" or parts.shape[-1] < 2:
            gs = parts.amax(-1)
        else:
            two = torch.topk(parts, 2, dim=-1).values
            gs = two[..., 0] + two[..., 1]
        best = torch.sort(gs, dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros_like(gs, dtype=torch.bool).scatter_(1, best, True)
        keep = keep.repeat_interleave(E // c["groups"], dim=1)
        adj = adj.masked_fill(~keep, float("-inf"))
    ids = torch.sort(adj, dim=-1, descending=True, stable=True).indices[:, :K]
    w = score.gather(1, ids)
    if c["renorm"] != "none":
        w = w / w.sum(-1, keepdim=True)
    return {"ids": ids.to(torch.int32), "weights": w * c["scale"]}


def _plain_delta(c, s):
    """Chunks of 32 tokens a sequence: inside a chunk the writes solve a unit lower triangular
    system (its inverse a product of log2 terms), between chunks the state carries over."""
    N, most = s["state"].shape[0], s["longest"]
    T, H, V = s["v"].shape
    K, r = s["q"].shape[-1], H // s["q"].shape[1]
    lens = s["offsets"][1:] - s["offsets"][:-1]
    if s["limits"] is not None:
        lens = torch.minimum(lens, s["limits"])
    C = min(32, most)
    steps = -(-most // C)
    at = torch.arange(steps * C, device=DEV)
    live = at < lens[:, None]
    idx = torch.where(live, s["offsets"][:-1, None] + at, 0).long()

    def rows(x):  # [N][H][steps * C][...], rows past a sequence's end zero
        y = x.float()[idx] * live.view(N, -1, *[1] * (x.dim() - 1))
        return y.transpose(1, 2)

    q, k, v = rows(s["q"]), rows(s["k"]), rows(s["v"])
    if c["norm"]:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + EPS)
    q, k = q.repeat_interleave(r, dim=1) * K ** -0.5, k.repeat_interleave(r, dim=1)
    beta = rows(s["beta"])[..., None]
    if s["gate"] is None:
        g = torch.zeros_like(beta)
    else:
        g = rows(s["gate"])
        g = g[..., None] if g.dim() == 3 else g
    S = s["state"]
    out = torch.zeros((N, steps * C, H, V), device=DEV)
    tri = torch.ones((C, C), dtype=torch.bool, device=DEV).tril()
    eye = torch.eye(C, device=DEV)
    for j in range(steps):
        w = slice(j * C, (j + 1) * C)
        G = torch.cumsum(g[:, :, w], 2)
        D = torch.exp((G[:, :, :, None] - G[:, :, None]).masked_fill(~tri[..., None],
                                                                     float("-inf")))
        kd = D * k[:, :, None, w]
        P = (q[:, :, w, None] * kd).sum(-1)
        A = beta[:, :, w] * (k[:, :, w, None] * kd).sum(-1).masked_fill(eye.bool(), 0.0)
        inv, power = eye - A, A @ A
        n = 2
        while n < C:
            inv, power, n = inv + inv @ power, power @ power, 2 * n
        carried = torch.exp(G)
        u = inv @ (beta[:, :, w] * (v[:, :, w] - (k[:, :, w] * carried) @ S))
        out[:, w] = ((q[:, :, w] * carried) @ S + P @ u).transpose(1, 2)
        last = G[:, :, -1:]
        S = S * torch.exp(last).transpose(2, 3) + \
            (k[:, :, w] * torch.exp(last - G)).transpose(2, 3) @ u
    flat = torch.zeros((T + 1, H, V), device=DEV)
    flat[torch.where(live, idx, T).reshape(-1)] = out.reshape(-1, H, V)
    return {"out": flat[:T].to(s["v"].dtype), "state": S}


def _plain_verify(c, s):
    target, tokens = s["target"], s["tokens"].long()
    N, D1, V = target.shape
    D = D1 - 1
    if c["greedy"]:
        t = target.float()
        at = torch.arange(V, device=DEV).expand_as(t)
        best = torch.where(t == t.amax(-1, keepdim=True), at, V).amin(-1)
        ok = best[:, :D] == tokens
        accepted = torch.cumprod(ok.long(), 1).sum(1)
        last = best.gather(1, accepted[:, None])
    else:
        def dist(x):  # 64 bits: sums over a vocabulary, tokens next to the border that u draws
            return x.double() if c["form"] == "probs" else \
                torch.softmax(x.double() / _f32(c["temperature"]), -1)
        p = dist(target)
        px = p[:, :D].gather(2, tokens[..., None])[..., 0]
        q = None if s["draft"] is None else dist(s["draft"])
        qx = 1.0 if q is None else q.gather(2, tokens[..., None])[..., 0]
        ok = s["accept_u"].double() * qx < px
        accepted = torch.cumprod(ok.long(), 1).sum(1)
        row = p[torch.arange(N, device=DEV), accepted]
        stop = accepted.clamp(max=D - 1)
        if q is None:
            other = torch.zeros_like(row).scatter_(1, tokens.gather(1, stop[:, None]), 2.0)
        else:
            other = q[torch.arange(N, device=DEV), stop]
        rest = (row - other * (accepted < D)[:, None]).clamp(min=0)
        cum = torch.cumsum(rest, 1)
        last = (cum <= s["sample_u"].double()[:, None] * cum[:, -1:]).sum(1, keepdim=True)
        last = last.clamp(max=V - 1)
    at = torch.arange(D1, device=DEV)
    out = torch.where(at < accepted[:, None], torch.nn.functional.pad(tokens, (0, 1)), -1)
    out = torch.where(at == accepted[:, None], last, out)
    return {"accepted": accepted.to(torch.int32), "tokens": out.to(torch.int32)}


def _f32(x):
    """A number as an fp32 parameter holds it."""
    return torch.tensor(x, dtype=torch.float32).item()


# ---- the framework's calls --------------------------------------------------------------------

def _own_route(c, s):
    k3x, ctx = _binding(), _context()
    params = k3x.make_route_params(
        c["tokens"], c["experts"], c["top_k"],
        scoring={"sigmoid": k3x.SCORE_SIGMOID, "softmax": k3x.SCORE_SOFTMAX}[c["scoring"]],
        renorm={"float": k3x.RENORM_FLOAT, "double": k3x.RENORM_DOUBLE,
                "none": k3x.RENORM_NONE}[c["renorm"]],
        routed_scale=c["scale"], groups=c["groups"], top_groups=c["top_groups"],
        group_score={"max": k3x.GROUP_MAX, "top2": k3x.GROUP_TOP2}[c["group_score"]])
    k3x.check(k3x.route(ctx, params, s["logits"], s["ids"], s["weights"], bias=s["bias"]), "route")
    return {"ids": s["ids"], "weights": s["weights"]}


def _own_delta(c, s):
    k3x, ctx = _binding(), _context()
    N = s["state"].shape[0]
    params = k3x.make_delta_params(s["q"], s["k"], s["v"], N, gate=s["gate"],
                                   scale=c["key_dim"] ** -0.5, norm_epsilon=EPS if c["norm"] else 0.0,
                                   longest=s["longest"])
    if "workspace" not in s:
        n = k3x.delta_workspace_bytes(params)
        s["workspace"] = torch.empty((n,), dtype=torch.uint8, device=DEV) if n else None
    k3x.check(k3x.delta_rule(ctx, params, s["q"], s["k"], s["v"], s["beta"], s["out"],
                             gate=s["gate"], offsets=s["offsets"], limits=s["limits"],
                             state_in=s["state"], state_out=s["state_out"],
                             workspace=s["workspace"]), "delta_rule")
    return {"out": s["out"], "state": s["state_out"]}


def _own_verify(c, s):
    k3x, ctx = _binding(), _context()
    params = k3x.make_verify_params(
        s["target"], form={"logits": k3x.DIST_LOGITS, "probs": k3x.DIST_PROBS}[c["form"]],
        greedy=c["greedy"], temperature=c["temperature"])
    if "workspace" not in s:
        n = k3x.verify_workspace_bytes(params)
        s["workspace"] = torch.empty((n,), dtype=torch.uint8, device=DEV) if n else None
    k3x.check(k3x.verify_draft(ctx, params, s["target"], s["tokens"], s["accepted"],
                               s["out_tokens"], draft=s["draft"],
                               accept_u=None if c["greedy"] else s["accept_u"],
                               sample_u=None if c["greedy"] else s["sample_u"],
                               workspace=s["workspace"]), "verify_draft")
    return {"accepted": s["accepted"], "tokens": s["out_tokens"]}


def run(s):
    c = s["case"]
    if own:
        return {"route": _own_route, "delta": _own_delta, "verify": _own_verify}[c["kind"]](c, s)
    return {"route": _plain_route, "delta": _plain_delta, "verify": _plain_verify}[c["kind"]](c, s)


# ---- 64 bits, from the definitions ------------------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "route":
        return _exact_route(c, s)
    if c["kind"] == "delta":
        return _exact_delta(c, s)
    return _exact_verify(c, s)


def _exact_route(c, s):
    """The choice goes by the rounded scores, so it is the definition's own; weights in 64 bits."""
    ids = _plain_route(c, s)["ids"].long()
    l = s["logits"].double()
    score = torch.sigmoid(l) if c["scoring"] == "sigmoid" else torch.softmax(l, -1)
    w = torch.gather(score, 1, ids)
    if c["renorm"] != "none":
        w = w / w.sum(1, keepdim=True)
    return {"ids": None, "weights": w * _f32(c["scale"])}


def _exact_delta(c, s):
    """Token by token, every sequence's t-th token at once."""
    lens = torch.tensor(_lens(c), device=DEV)
    if s["limits"] is not None:
        lens = torch.minimum(lens, s["limits"].long())
    start = s["offsets"][:-1].long()
    S = s["state"].double().clone()
    T, H, V = s["v"].shape
    K, r = s["q"].shape[-1], H // s["q"].shape[1]
    out = torch.zeros((T, H, V), dtype=torch.float64, device=DEV)
    scale = _f32(K ** -0.5)
    lens_host, start_host = lens.tolist(), start.tolist()
    for t in range(max(lens_host) if lens_host else 0):
        who = [n for n, most in enumerate(lens_host) if t < most]
        w = torch.tensor(who, device=DEV)
        rows = torch.tensor([start_host[n] + t for n in who], device=DEV)
        q, k, v = (s[x][rows].double() for x in "qkv")
        if c["norm"]:
            q = q * (q.square().sum(-1, keepdim=True) + EPS).rsqrt()
            k = k * (k.square().sum(-1, keepdim=True) + EPS).rsqrt()
        head = torch.arange(H, device=DEV) // r
        q, k = q[:, head] * scale, k[:, head]
        M = S[w]
        if s["gate"] is not None:
            decay = s["gate"][rows].double().exp()
            M = M * (decay[..., None] if decay.dim() == 3 else decay[..., None, None])
        u = s["beta"][rows].double()[..., None] * (v - (M * k[..., None]).sum(2))
        M = M + k[..., None] * u[:, :, None]
        out[rows] = (M * q[..., None]).sum(2)
        S[w] = M
    return {"out": out, "state": S}


def _exact_verify(c, s):
    """One sequence after another, as the definition reads."""
    N, D, V = c["sequences"], c["drafts"], c["vocab"]
    accepted = torch.zeros(N, dtype=torch.int32)
    tokens = torch.full((N, D + 1), -1, dtype=torch.int32)

    def dist(row):
        if c["form"] == "probs":
            return row.double()
        e = row.double() / _f32(c["temperature"])
        e = (e - e.max()).exp()
        return e / e.sum()

    for n in range(N):
        i = 0
        while i < D:
            x = int(s["tokens"][n, i])
            if c["greedy"]:
                row = s["target"][n, i].float()
                if int((row == row.max()).nonzero()[0]) != x:
                    break
            else:
                p = dist(s["target"][n, i])
                q = 1.0 if s["draft"] is None else float(dist(s["draft"][n, i])[x])
                if not float(s["accept_u"][n, i]) * q < float(p[x]):
                    break
            tokens[n, i] = x
            i += 1
        accepted[n] = i
        if c["greedy"]:
            row = s["target"][n, i].float()
            tokens[n, i] = int((row == row.max()).nonzero()[0])
            continue
        rest = dist(s["target"][n, i])
        if i < D:
            if s["draft"] is None:
                rest = rest.clone()
                rest[int(s["tokens"][n, i])] = 0
            else:
                rest = (rest - dist(s["draft"][n, i])).clamp(min=0)
        cum = rest.cumsum(0)
        tokens[n, i] = int((cum > float(s["sample_u"][n]) * cum[-1]).nonzero()[0])
    return {"accepted": accepted, "tokens": tokens}
