"""The feed-forward operators that are measured, with their plain forms.

  gated           H = act(X Wg^T) * (X Wu^T), optionally with G = X Wg^T and U = X Wu^T kept for the gradient
  gated_backward  dX, dWg, dWu of it from dH, X, Wg, Wu, G, U
  w4_nt           Y = X W^T with W[n, k] = s[k // group, n] * (q[n, k] - 8) held in 4 bits
  w4_gated        the gated form with both weights in 4 bits
  w4_quantize     bf16 weights into 4-bit codes and group scales, and back into the values that they stand for

Activations and weights are bf16, row-major; codes are bytes [N, K / 2] with the even k in the low four bits; scales are
bf16 [K / group, N].
"""
import math

import torch

own = False

DEV = "cuda:0"
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "none")


def listed():
    return [
        # one token through a gated block of the repository's MLP sizes: the weights are all that moves
        {"name": "gated 1x14336x4096", "op": "gated", "M": 1, "F": 14336, "K": 4096, "act": "silu", "save": False},
        # a few sequences decoded together, a block whose width divides by nothing
        {"name": "gated 23x5003x2056", "op": "gated", "M": 23, "F": 5003, "K": 2056, "act": "gelu", "save": False},
        # a short prompt with an odd number of tokens
        {"name": "gated 777x5120x2048", "op": "gated", "M": 777, "F": 5120, "K": 2048, "act": "gelu_tanh", "save": False},
        # the forward half of a training step, G and U kept for the gradient
        {"name": "gated 8192x14336x4096 save", "op": "gated", "M": 8192, "F": 14336, "K": 4096, "act": "silu", "save": True},
        # gradients of a small block on a ragged batch
        {"name": "backward 333x1003x520", "op": "gated_backward", "M": 333, "F": 1003, "K": 520, "act": "gelu"},
        # gradients of an ordinary micro-batch
        {"name": "backward 2048x8192x2048", "op": "gated_backward", "M": 2048, "F": 8192, "K": 2048, "act": "silu"},
        # gradients of the block at the repository's MLP sizes
        {"name": "backward 8192x14336x4096", "op": "gated_backward", "M": 8192, "F": 14336, "K": 4096, "act": "silu"},
        # one token through a down projection with 4-bit weights
        {"name": "w4 1x4096x14336 g128", "op": "w4_nt", "M": 1, "N": 4096, "K": 14336, "group": 128},
        # a batch of tokens through a wide 4-bit projection
        {"name": "w4 32x8192x8192 g64", "op": "w4_nt", "M": 32, "N": 8192, "K": 8192, "group": 64},
        # a few tokens through a 4-bit gated block, fine groups, an odd width
        {"name": "w4 gated 5x14331x4096 g32", "op": "w4_gated", "M": 5, "N": 14331, "K": 4096, "group": 32, "act": "silu"},
        # weights of one MLP projection quantised for serving
        {"name": "w4 quantize 14336x4096 g128", "op": "w4_quantize", "N": 14336, "K": 4096, "group": 128},
        # the same for an odd, small projection with fine groups
        {"name": "w4 quantize 1001x2080 g32", "op": "w4_quantize", "N": 1001, "K": 2080, "group": 32},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("gated", "gated", "gated_backward", "gated_backward", "w4_nt", "w4_nt", "w4_gated", "w4_quantize"))
    if op in ("gated", "gated_backward"):
        while True:
            M = _log(rng, 1, 8192)
            F = _log(rng, 256, 14336)
            K = 8 * _log(rng, 32, 1024)
            if M * F * K <= 8192 * 14336 * 4096:
                break
        case = {"op": op, "M": M, "F": F, "K": K, "act": rng.choice(ACTS)}
        if op == "gated":
            case["save"] = rng.random() < 0.5
        return case
    group = rng.choice((32, 64, 128, 256))
    K = group * max(1, _log(rng, 512, 14336) // group)
    N = _log(rng, 256, 14336)
    if op == "w4_quantize":
        return {"op": op, "N": N, "K": K, "group": group}
    case = {"op": op, "M": _log(rng, 1, 32), "N": N, "K": K, "group": group}
    if op == "w4_gated":
        case["act"] = rng.choice(ACTS)
    return case


def _rows(M, N, g, std):
    """A bf16 [M, N] matrix whose rows start on 16-byte boundaries, as activations are kept where N is odd."""
    pitch = 8 * ((N + 7) // 8)
    return (torch.randn(M, pitch, generator=g, device=DEV) * std).to(torch.bfloat16)[:, :N]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    op = case["op"]
    s = {"op": op, "act": case.get("act")}
    if op in ("gated", "gated_backward"):
        M, F, K = case["M"], case["F"], case["K"]
        s["x"] = _rows(M, K, g, 1.0)
        s["wg"], s["wu"] = (_rows(F, K, g, K ** -0.5) for _ in range(2))
        s["save"] = case.get("save", False)
        if op == "gated_backward":
            s["g"], s["u"] = (_rows(M, F, g, 1.0) for _ in range(2))
            s["dh"] = _rows(M, F, g, 0.05)
        return s
    N, K, group = case["N"], case["K"], case["group"]
    s["group"] = group
    if op == "w4_quantize":
        s["w"] = _rows(N, K, g, K ** -0.5)
        return s
    s["x"] = _rows(case["M"], K, g, 1.0)
    for name in ("gate", "up") if op == "w4_gated" else ("w",):
        codes = torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
        spread = torch.randn(K // group, N, generator=g, device=DEV) * 0.3
        s[name] = (codes, (spread.exp() * (K ** -0.5 / 4.6)).to(torch.bfloat16))
    return s


# ------------------------------------------------------------- plain forms


def _act(x, kind):
    if kind == "silu":
        return x / (1.0 + torch.exp(-x))
    if kind == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * 0.5 ** 0.5))
    if kind == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (x + 0.044715 * x * x * x)))
    if kind == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    return x


def _act_grad(x, kind):
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-x))
        return s * (1.0 + x * (1.0 - s))
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(x * 0.5 ** 0.5)) + x * torch.exp(-0.5 * x * x) * (0.5 / math.pi) ** 0.5
    if kind == "gelu_tanh":
        c = (2.0 / math.pi) ** 0.5
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * x * x)
    if kind == "relu":
        return (x > 0).to(x.dtype)
    return torch.ones_like(x)


def _w4_values(codes, scales, group):
    low, high = codes & 15, codes >> 4
    q = torch.stack((low, high), dim=-1).reshape(codes.shape[0], -1).float() - 8.0
    return q * scales.float().t().repeat_interleave(group, dim=1)


def _plain(s):
    op = s["op"]
    if op == "gated":
        x = s["x"].float()
        g, u = x @ s["wg"].float().t(), x @ s["wu"].float().t()
        h = (_act(g, s["act"]) * u).bfloat16()
        return {"h": h, "g": g.bfloat16(), "u": u.bfloat16()} if s["save"] else {"h": h}
    if op == "gated_backward":
        x, dh, g, u = s["x"].float(), s["dh"].float(), s["g"].float(), s["u"].float()
        du = dh * _act(g, s["act"])
        dg = dh * u * _act_grad(g, s["act"])
        dx = dg @ s["wg"].float() + du @ s["wu"].float()
        return {"dx": dx.bfloat16(), "dwg": (dg.t() @ x).bfloat16(), "dwu": (du.t() @ x).bfloat16()}
    if op == "w4_nt":
        return {"y": (s["x"].float() @ _w4_values(*s["w"], s["group"]).t()).bfloat16()}
    if op == "w4_gated":
        x = s["x"].float()
        g, u = (x @ _w4_values(*s[name], s["group"]).t() for name in ("gate", "up"))
        return {"h": (_act(g, s["act"]) * u).bfloat16()}
    w, group = s["w"].float(), s["group"]
    blocks = w.reshape(w.shape[0], -1, group)
    scales = (blocks.abs().amax(dim=2) / 7.0).bfloat16()
    f = scales.float().unsqueeze(2)
    q = torch.where(f > 0, torch.round(blocks / f), torch.zeros_like(blocks)).clamp(-8.0, 7.0)
    return {"scales": scales.t().contiguous(), "values": (q * f).reshape(w.shape).bfloat16()}


def _own(s):
    import b200_gemm_b200 as b200

    op = s["op"]
    if op == "gated":
        if s["save"]:
            h, g, u = b200.gated(s["x"], s["wg"], s["wu"], activation=s["act"], save=True)
            return {"h": h, "g": g, "u": u}
        return {"h": b200.gated(s["x"], s["wg"], s["wu"], activation=s["act"])}
    if op == "gated_backward":
        dx, dwg, dwu = b200.gated_backward(s["dh"], s["x"], s["wg"], s["wu"], s["g"], s["u"], activation=s["act"])
        return {"dx": dx, "dwg": dwg, "dwu": dwu}
    if op == "w4_nt":
        return {"y": b200.w4_nt(s["x"], *s["w"])}
    if op == "w4_gated":
        return {"h": b200.w4_gated(s["x"], *s["gate"], *s["up"], activation=s["act"])}
    codes, scales = b200.w4_quantize(s["w"], group=s["group"])
    return {"scales": scales, "values": b200.w4_dequantize(codes, scales)}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    op = case["op"]
    if op in ("gated", "gated_backward"):
        M, F, K = case["M"], case["F"], case["K"]
        if op == "gated":
            return {"bytes": 2 * (M * K + 2 * F * K + M * F * (3 if case["save"] else 1)), "flops": 4 * M * F * K}
        return {"bytes": 2 * (3 * M * F + 2 * M * K + 4 * F * K), "flops": 8 * M * F * K}
    N, K, group = case["N"], case["K"], case["group"]
    if op == "w4_quantize":
        return {"bytes": 4 * N * K + 2 * N * (K // group), "flops": 4 * N * K}
    sides = 2 if op == "w4_gated" else 1
    M = case["M"]
    return {"bytes": sides * (N * K // 2 + 2 * N * (K // group)) + 2 * M * (K + N), "flops": 2 * sides * M * N * K}


# ------------------------------------------------------- in 64 bits, apart


def _phi(x):
    """The normal distribution's integral, by the complement so that its lower tail keeps its digits."""
    return 0.5 * torch.special.erfc(-x / math.sqrt(2.0))


def _exact_act(x, kind):
    """The activation and its derivative."""
    if kind == "silu":
        s = torch.sigmoid(x)
        return x * s, s + x * s * torch.sigmoid(-x)
    if kind == "gelu":
        return x * _phi(x), _phi(x) + x * torch.exp(-x * x / 2.0) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":  # (1 + tanh z) / 2 is the logistic function of 2 z
        z = math.sqrt(8.0 / math.pi) * x * (1.0 + 0.044715 * x.square())
        s = torch.sigmoid(z)
        return x * s, s + x * s * torch.sigmoid(-z) * math.sqrt(8.0 / math.pi) * (1.0 + 0.134145 * x.square())
    if kind == "relu":
        return x.clamp(min=0.0), (x > 0).double()
    return x, torch.ones_like(x)


def _exact_w4(pair, group):
    codes, scales = pair
    N, K = codes.shape[0], 2 * codes.shape[1]
    w = torch.empty(N, K, dtype=torch.float64, device=codes.device)
    w[:, 0::2] = torch.remainder(codes, 16).double() - 8.0
    w[:, 1::2] = torch.div(codes, 16, rounding_mode="floor").double() - 8.0
    return (w.view(N, K // group, group) * scales.double().t().unsqueeze(2)).view(N, K)


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "gated":
        x = s["x"].double()
        g, u = torch.mm(x, s["wg"].double().t()), torch.mm(x, s["wu"].double().t())
        h = _exact_act(g, s["act"])[0].mul_(u)
        return {"h": h, "g": g, "u": u} if s["save"] else {"h": h}
    if op == "gated_backward":
        a, da = _exact_act(s["g"].double(), s["act"])
        dh, x = s["dh"].double(), s["x"].double()
        du = a.mul_(dh)
        dg = da.mul_(dh).mul_(s["u"].double())
        dx = torch.addmm(torch.mm(dg, s["wg"].double()), du, s["wu"].double())
        return {"dx": dx, "dwg": torch.mm(dg.t(), x), "dwu": torch.mm(du.t(), x)}
    if op == "w4_nt":
        return {"y": torch.mm(s["x"].double(), _exact_w4(s["w"], s["group"]).t())}
    if op == "w4_gated":
        x = s["x"].double()
        g, u = (torch.mm(x, _exact_w4(s[name], s["group"]).t()) for name in ("gate", "up"))
        return {"h": _exact_act(g, s["act"])[0] * u}
    w = s["w"].double().view(case["N"], -1, s["group"])
    scales = (w.abs().max(dim=2).values / 7.0).to(torch.bfloat16).double()
    step = scales.unsqueeze(2).expand_as(w)
    q = torch.zeros_like(w)
    q[step > 0] = (w[step > 0] / step[step > 0]).round().clamp(-8, 7)
    return {"scales": scales.t().contiguous(), "values": (q * step).view(case["N"], -1)}
