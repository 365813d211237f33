"""Operator cases: row operations over the vocabulary that distil one model into another and check what the second one drafts.

    top      the k largest logits of a row with their log-probabilities, and the row's log-sum-exp (what a teacher hands on)
    distill  the divergence of a student's row from a teacher's top logits, and its gradient
    softmax  a row's probabilities at a temperature
    verify   which drafted tokens stand against the target's probabilities, and the token that follows them, from given random numbers

A row is the logits (or probabilities) of one position over the whole vocabulary.  Formulas, for a row z and a temperature T:

    s_v = z_v / T - log sum_u exp(z_u / T),  p_v = exp(s_v)
    top      the k largest z (ties: the lowest index first), their s, and log sum exp(z / T)
    distill  from entries (i_j, t_j), t_j a teacher's log-probability of index i_j, no entry where i_j = -1:
             "renorm"  q_j = exp(t_j) / sum exp(t);  loss = sum q_j (log q_j - s_{i_j});  d/dz_v = (p_v - q_v) / T
             "tail"    q_j = exp(t_j), r = max(0, 1 - sum q), R = sum of p over the indices not listed;
                       loss = sum q_j (t_j - s_{i_j}) + r (log r - log R);
                       d/dz_v = (p_v - q_v) / T for a listed v, p_v (1 - r / R) / T for the others
             both times the row's weight w; f16 gradients come without the factor w / T, which is returned beside them
    verify   drafted token d_i stands if all before it do and u_i q_i(d_i) < p_i(d_i) (q = 1 for drafts without probabilities);
             behind the last one that stands a token is drawn with u from max(p - q, 0) at the first that does not (p without
             that token, for drafts without probabilities), or from p of the position behind the last: the lowest index whose
             running sum exceeds u times the whole sum
"""
from __future__ import annotations

import random

import torch

own = False  # False: the plain forms below; True: the package's operators

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}
MODES = {"renorm": 0, "tail": 1}

# ------------------------------------------------------------------ the cases


def listed() -> list:
    return [
        # One position's teacher logits: latency is all of it.
        dict(name="top-8-of-151936-f32-x1", kind="top", rows=1, vocab=151936, pad=0, dtype="f32", temperature=1.0, k=8),
        # What a model's head hands over at once: 1024 rows of f32 logits.
        dict(name="top-64-of-151936-f32-x1024", kind="top", rows=1024, vocab=151936, pad=0, dtype="f32", temperature=1.0, k=64),
        # A host that keeps its teacher's logits in 16 bits, softened: values of bf16 tie often.
        dict(name="top-32-of-128256-bf16-x4096", kind="top", rows=4096, vocab=128256, pad=0, dtype="bf16", temperature=2.0, k=32),
        # A test-sized model: rows of 640, a few entries each, the teacher's rest as one bucket.
        dict(name="distill-tail-5-of-640-f32-x37", kind="distill", rows=37, vocab=640, pad=0, dtype="f32", out="f32", temperature=1.0,
             k=5, mode="tail", short=True),
        # The distillation step of the model driver: 1024 rows of f32 logits, gradients as f16 rows with a factor each.
        dict(name="distill-64-of-151936-f32-x1024", kind="distill", rows=1024, vocab=151936, pad=0, dtype="f32", out="f16", temperature=1.0,
             k=64, mode="renorm", short=False),
        # The largest: 16-bit logits of a host's own head and gradients for it, softened, with the rest as a bucket.
        dict(name="distill-tail-32-of-128256-bf16-x2048", kind="distill", rows=2048, vocab=128256, pad=0, dtype="bf16", out="bf16",
             temperature=2.0, k=32, mode="tail", short=False),
        # The loss alone, as an evaluation wants it, over an odd vocabulary in padded rows.
        dict(name="distill-loss-16-of-50021-f16-x777", kind="distill", rows=777, vocab=50021, pad=27, dtype="f16", out="none",
             temperature=1.0, k=16, mode="tail", short=True),
        # The probabilities of one drafted run: four drafted positions and the one behind them.
        dict(name="softmax-151936-f32-x5", kind="softmax", rows=5, vocab=151936, pad=0, dtype="f32", out="f32", temperature=0.7),
        # Those of a large batch from 16-bit logits.
        dict(name="softmax-128256-bf16-x1536", kind="softmax", rows=1536, vocab=128256, pad=0, dtype="bf16", out="f32", temperature=1.0),
        # One sequence, four drafted tokens: the smallest check.
        dict(name="verify-1x4-of-151936-f32", kind="verify", n_seq=1, max_draft=4, ragged=False, vocab=151936, pad=0, dtype="f32", draft_prob=True),
        # Many sequences with up to eight drafted tokens each, probabilities in 16 bits.
        dict(name="verify-96x8-of-128256-bf16", kind="verify", n_seq=96, max_draft=8, ragged=True, vocab=128256, pad=0, dtype="bf16", draft_prob=True),
        # Drafts that come without probabilities (copied from a prompt, or another model's greedy tokens).
        dict(name="verify-32x3-of-151936-f32-greedy", kind="verify", n_seq=32, max_draft=3, ragged=True, vocab=151936, pad=0, dtype="f32", draft_prob=False),
    ]


#: Row elements of a drawn case at most: those of the largest listed ones of its kind.
MOST = {"top": 4096 * 128256, "distill": 2048 * 128256, "softmax": 1536 * 128256, "verify": 96 * 9 * 128256}
VOCABS = (151936, 128256)  # of the models this package knows


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["top", "distill", "distill", "softmax", "verify"])
    vocab = rng.choice(VOCABS) if rng.random() < 0.3 else _log_int(rng, 200, 262144)
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    case = dict(kind=kind, vocab=vocab, pad=rng.choice([0, 0, rng.randint(1, 64)]), dtype=dtype)
    if kind == "verify":
        max_draft = rng.randint(1, 12)
        n_seq = _log_int(rng, 1, max(1, min(256, MOST[kind] // (2 * (max_draft + 1) * vocab))))
        return dict(case, n_seq=n_seq, max_draft=max_draft, ragged=rng.random() < 0.6, draft_prob=rng.random() < 0.7)
    rows = _log_int(rng, 1, max(1, min(4096, MOST[kind] // vocab)))
    case = dict(case, rows=rows, temperature=rng.choice([1.0, 1.0, 2.0, 0.7, 4.0]))
    if kind == "softmax":
        return dict(case, out=rng.choice(["f32", dtype]))
    k = _log_int(rng, 1, min(128, vocab))
    if kind == "top":
        return dict(case, k=k)
    return dict(case, out=rng.choice(["f32", "f16", dtype, dtype, "none"]), k=k, mode=rng.choice(["renorm", "tail"]), short=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs


class _State:
    pass


def _padded(x: torch.Tensor, pad: int) -> torch.Tensor:
    """x with `pad` columns of NaN behind every row: a user's rows may be longer than the vocabulary."""
    return torch.nn.functional.pad(x, (0, pad), value=float("nan")) if pad else x


def _logits(rows: int, vocab: int, gen) -> torch.Tensor:
    """Logits as a trained model has them: the largest of a row holds a tenth of its mass or so."""
    return torch.randn(rows, vocab, generator=gen, device="cuda").mul_(2.5)


def prepare(case: dict, seed: int):
    s = _State()
    s.case = case
    gen = torch.Generator("cuda").manual_seed(seed)
    vocab, t = case["vocab"], TYPES[case["dtype"]]
    if case["kind"] == "verify":
        _prepare_verify(s, case, seed, gen)
        return s
    rows = case["rows"]
    z = _logits(rows, vocab, gen)
    s.logits = _padded(z.to(t), case["pad"])
    if case["kind"] == "top":
        s.index = torch.empty(rows, case["k"], dtype=torch.int32, device="cuda")
        s.logp = torch.empty(rows, case["k"], device="cuda")
        s.lse = torch.empty(rows, device="cuda")
    elif case["kind"] == "softmax":
        s.prob = torch.empty(rows, vocab, dtype=TYPES[case["out"]], device="cuda")
    else:  # a teacher that agrees with the student in part
        k, temperature = case["k"], case["temperature"]
        z = z.add(torch.randn(z.shape, generator=gen, device="cuda")).div_(temperature)  # the logits may be z itself
        top = z.topk(k, dim=1)
        s.index = top.indices.to(torch.int32)
        s.teacher = top.values - z.logsumexp(1, keepdim=True)
        if case["short"]:  # rows with fewer entries than k, one row in nine without any
            n = torch.randint(0, k + 1, (rows, 1), generator=gen, device="cuda")
            n[::9] = 0
            s.index[torch.arange(k, device="cuda") >= n] = -1
        s.weight = torch.rand(rows, generator=gen, device="cuda").add_(0.5).div_(rows)
        s.loss = torch.empty(rows, device="cuda")
        if case["out"] != "none":
            s.grad = torch.empty(rows, vocab, dtype=TYPES[case["out"]], device="cuda")
        if case["out"] == "f16":
            s.factor = torch.empty(rows, device="cuda")
    return s


def _prepare_verify(s, case: dict, seed: int, gen) -> None:
    rng = random.Random(seed)
    n_seq, vocab, t = case["n_seq"], case["vocab"], TYPES[case["dtype"]]
    shape = random.Random(f"{n_seq} {case['max_draft']}")  # how many tokens each sequence drafts is part of the case
    counts = [shape.randint(0, case["max_draft"]) if case["ragged"] else case["max_draft"] for _ in range(n_seq)]
    counts[rng.randrange(n_seq) if case["ragged"] else 0] = case["max_draft"]
    starts = [sum(counts[:i]) for i in range(n_seq + 1)]
    total = starts[-1]
    z = _logits(total + n_seq, vocab, gen)
    s.target = _padded(z.softmax(1).to(t), case["pad"])
    drafted = [starts[i] + i + j for i in range(n_seq) for j in range(counts[i])]
    zq = z[torch.tensor(drafted, dtype=torch.long, device="cuda")]
    zq.add_(torch.randn(zq.shape, generator=gen, device="cuda"), alpha=0.7)  # a smaller model's
    q = zq.softmax(1).to(t)
    if case["draft_prob"]:
        s.draft = _padded(q, case["pad"])
        s.tokens = torch.multinomial(q.float(), 1, generator=gen)[:, 0].to(torch.int32)
    else:
        s.draft = None
        s.tokens = q.argmax(1).to(torch.int32)
    s.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s.u_accept = torch.rand(total, generator=gen, device="cuda")
    s.u_sample = torch.rand(n_seq, generator=gen, device="cuda")
    s.accepted = torch.empty(n_seq, dtype=torch.int32, device="cuda")
    s.token = torch.empty(n_seq, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ one pass

_CTX = None


def _ctx():
    """One context per process, as a program keeps it, on torch's stream."""
    global _CTX
    if _CTX is None:
        import rust_trainer_b200 as rt

        _CTX = rt.Context(0)
        _CTX.check(rt.lib().rt_ctx_set_stream(_CTX._h, torch.cuda.current_stream().cuda_stream))
        _CTX.L = rt.lib()
    return _CTX


def run(s):
    kind = s.case["kind"]
    if own:
        return _run_own(s, kind)
    if kind == "top":
        return _top_plain(s)
    if kind == "softmax":
        return _softmax_plain(s)
    if kind == "distill":
        return _distill_plain(s)
    return _verify_plain(s)


def _run_own(s, kind: str):
    c, case = _ctx(), s.case
    L, h, t = c.L, c._h, CODES[case["dtype"]]
    if kind == "verify":
        q = s.draft
        c.check(L.rt_verify_draft_dev(h, s.target.data_ptr(), s.target.stride(0), None if q is None else q.data_ptr(), 0 if q is None else q.stride(0),
                                      t, case["vocab"], s.tokens.data_ptr(), s.starts.data_ptr(), case["n_seq"], s.tokens.numel(),
                                      s.u_accept.data_ptr(), s.u_sample.data_ptr(), s.accepted.data_ptr(), s.token.data_ptr()))
        return {"accepted": s.accepted, "token": s.token}
    z, rows, vocab = s.logits, case["rows"], case["vocab"]
    if kind == "top":
        c.check(L.rt_top_logits_dev(h, z.data_ptr(), t, rows, vocab, z.stride(0), case["temperature"], case["k"], s.index.data_ptr(),
                                    s.logp.data_ptr(), s.lse.data_ptr()))
        return {"index": s.index, "logp": s.logp, "lse": s.lse}
    if kind == "softmax":
        c.check(L.rt_softmax_dev(h, z.data_ptr(), t, rows, vocab, z.stride(0), case["temperature"], s.prob.data_ptr(), CODES[case["out"]], vocab))
        return {"prob": s.prob}
    out = case["out"]
    grad = None if out == "none" else s.grad.data_ptr()
    factor = s.factor.data_ptr() if out == "f16" else None
    c.check(L.rt_distill_dev(h, z.data_ptr(), t, rows, vocab, z.stride(0), case["temperature"], s.index.data_ptr(), s.teacher.data_ptr(), case["k"],
                             MODES[case["mode"]], s.weight.data_ptr(), s.loss.data_ptr(), grad, CODES.get(out, 0), vocab, factor))
    return _distill_outputs(s, s.loss, None if out == "none" else s.grad, s.factor if out == "f16" else None)


def _distill_outputs(s, loss, grad, factor):
    got = {"loss": loss}
    if grad is not None:
        got["grad"] = grad
    if factor is not None:
        got["factor"] = factor
    return got


def _shifted(s):
    """(z - max) / T in f32."""
    z = s.logits[:, :s.case["vocab"]].float()
    m = z.amax(1, keepdim=True)
    return (z - m).div_(s.case["temperature"]), m


def _top_plain(s):
    x, m = _shifted(s)
    vocab, k = s.case["vocab"], s.case["k"]
    bits = (s.logits[:, :vocab].float() + 0.0).view(torch.int32)  # + 0: the two zeros tie
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()  # integers in the order of the values
    key = (order << 32) + torch.arange(vocab - 1, -1, -1, device=x.device)
    index = key.topk(k, dim=1).indices
    log_sum = x.exp().sum(1, keepdim=True).log()
    return {"index": index.to(torch.int32), "logp": x.gather(1, index) - log_sum, "lse": (m / s.case["temperature"] + log_sum)[:, 0]}


def _softmax_plain(s):
    e = _shifted(s)[0].exp_()
    return {"prob": (e / e.sum(1, keepdim=True)).to(TYPES[s.case["out"]])}


def _distill_plain(s):
    case = s.case
    x, m = _shifted(s)
    entry = s.index >= 0
    at = s.index.long().clamp(min=0)
    e = x.exp_()
    total = e.sum(1, keepdim=True, dtype=torch.float64)  # the loss is a small difference of large terms
    log_p = (s.logits.gather(1, at).double() - m.double()) / case["temperature"] - total.log()
    t = s.teacher.double().masked_fill(~entry, -torch.inf)
    q = t.exp()  # few values a row, and what is left beside their sum
    share = 1.0 / total
    if case["mode"] == "renorm":
        mass = q.sum(1, keepdim=True)
        q = torch.where(mass > 0, q / mass, 0.0)
        loss = torch.where(q > 0, q * (q.log() - log_p), 0.0).sum(1)
        share_rest = share
    else:
        r = (1.0 - q.sum(1, keepdim=True)).clamp(min=0)
        rest = e.scatter(1, torch.where(entry, at, at[:, :1]), 0.0)  # an empty place repeats the row's first, if it has one
        rest = torch.where(entry[:, :1], rest.sum(1, keepdim=True, dtype=torch.float64), total)
        loss = torch.where(q > 0, q * (t - log_p), 0.0).sum(1)
        loss = loss + torch.where(r > 0, r * (r.log() - (rest / total).log()), 0.0)[:, 0]
        share_rest = share - r / rest
    loss = (s.weight * loss).float()
    if case["mode"] == "renorm":  # rows without entries have nothing to learn from
        share = share_rest = torch.where(mass > 0, share, 0.0)
    if case["out"] == "none":
        return _distill_outputs(s, loss, None, None)
    grad = torch.empty(e.shape[0], e.shape[1] + 1, device=e.device)  # the last column takes what empty places write
    torch.mul(e, share_rest.float(), out=grad[:, :-1])
    grad.scatter_(1, torch.where(entry, at, e.shape[1]), (e.gather(1, at) * share - q).float())
    grad = grad[:, :-1]
    factor = s.weight / case["temperature"]
    if case["out"] == "f16":
        return _distill_outputs(s, loss, grad.to(torch.float16), factor)
    return _distill_outputs(s, loss, (grad * factor[:, None]).to(TYPES[case["out"]]), None)


def _verify_plain(s):
    case = s.case
    vocab, n = case["vocab"], s.tokens.numel()
    first, end = s.starts[:-1].long(), s.starts[1:].long()
    seq = torch.arange(case["n_seq"], device=first.device)
    at = first[:, None] + torch.arange(case["max_draft"], device=first.device)  # [sequence, draft]
    real = at < end[:, None]
    at = at.clamp(max=n - 1)
    tok = s.tokens[at].long()
    row = torch.where(real, at + seq[:, None], 0)
    p = s.target[row, tok].double()
    q = torch.ones_like(p) if s.draft is None else s.draft[at, tok].double()
    stands = real & (s.u_accept[at].double() * q < p)
    accepted = stands.long().cumprod(1).sum(1)
    whole = first + accepted == end
    p_row = s.target[first + seq + accepted, :vocab].double()
    at_reject = (first + accepted).clamp(max=n - 1)
    if s.draft is None:
        left = p_row.scatter(1, s.tokens[at_reject].long()[:, None], 0.0)
    else:
        left = (p_row - s.draft[at_reject, :vocab].double()).clamp(min=0)
    left = torch.where(whole[:, None] | (left.sum(1, keepdim=True) == 0), p_row, left)
    running = left.cumsum(1)
    token = (running <= s.u_sample.double()[:, None] * running[:, -1:]).sum(1)
    return {"accepted": accepted.to(torch.int32), "token": token.to(torch.int32)}


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "verify":
        return _verify_exact(s)
    parts = []
    step = max(1, (1 << 28) // case["vocab"])
    for lo in range(0, case["rows"], step):
        z = s.logits[lo:lo + step, :case["vocab"]].double()
        parts.append({"top": _top_exact, "softmax": _softmax_exact, "distill": _distill_exact}[case["kind"]](s, slice(lo, lo + step), z))
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def _top_exact(s, rows, z):
    value, index = z.sort(dim=1, descending=True, stable=True)
    lse = torch.logsumexp(z / s.case["temperature"], 1)
    k = s.case["k"]
    return {"index": index[:, :k].to(torch.int32), "logp": value[:, :k] / s.case["temperature"] - lse[:, None], "lse": lse}


def _softmax_exact(s, rows, z):
    return {"prob": torch.softmax(z / s.case["temperature"], 1)}


def _distill_exact(s, rows, z):
    case = s.case
    log_p = torch.log_softmax(z / case["temperature"], 1)
    q = torch.zeros_like(log_p)
    index, t = s.index[rows].cpu(), s.teacher[rows].double()
    row, j = (index >= 0).nonzero(as_tuple=True)
    row, j = row.cuda(), j.cuda()
    v = s.index[rows][row, j].long()
    q[row, v] = t[row, j].exp()
    listed = torch.zeros_like(q, dtype=torch.bool)
    listed[row, v] = True
    p = log_p.exp()
    if case["mode"] == "renorm":
        mass = q.sum(1, keepdim=True)
        empty = mass == 0
        q = q / mass.masked_fill(empty, 1.0)
        loss = (torch.xlogy(q, q) - q * log_p).sum(1)
        grad = (p - q).masked_fill(empty, 0.0)
    else:
        r = (1 - q.sum(1)).clamp(min=0)
        rest = p.masked_fill(listed, 0.0).sum(1)
        loss = (torch.xlogy(q, q) - q * log_p).sum(1) + torch.xlogy(r, r) - torch.where(r > 0, r * rest.log(), 0.0)
        grad = torch.where(listed, p - q, p * (1 - r / rest)[:, None])
    w = s.weight[rows].double()
    factor = w / case["temperature"]
    got = {"loss": w * loss}
    if case["out"] == "f16":
        got |= {"grad": grad, "factor": factor}
    elif case["out"] != "none":
        got["grad"] = grad * factor[:, None]
    return got


def _verify_exact(s):
    case, starts = s.case, s.starts.tolist()
    u, u_last, tokens = s.u_accept.double().tolist(), s.u_sample.double().tolist(), s.tokens.tolist()
    accepted, token = [], []
    for i in range(case["n_seq"]):
        n, left = 0, None
        for j in range(starts[i], starts[i + 1]):
            d = tokens[j]
            p = s.target[j + i, :case["vocab"]].double()
            q = torch.zeros_like(p) if s.draft is None else s.draft[j, :case["vocab"]].double()
            if s.draft is None:
                q[d] = 1.0
            if u[j] * float(q[d]) < float(p[d]):
                n += 1
                continue
            left = torch.relu(p - q)
            if float(left.sum()) == 0.0:
                left = p
            break
        if left is None:
            left = s.target[starts[i + 1] + i, :case["vocab"]].double()
        sums = torch.cumsum(left, 0)
        accepted.append(n)
        token.append(int(torch.searchsorted(sums, u_last[i] * sums[-1], right=True)))
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "token": torch.tensor(token, dtype=torch.int32)}


# ------------------------------------------------------------------ what no implementation can do without


def work(case: dict) -> dict:
    size = {"f32": 4, "bf16": 2, "f16": 2, "none": 0}
    vocab, e = case["vocab"], size[case["dtype"]]
    if case["kind"] == "verify":
        # one row of the target's for each sequence, and one of the draft's where a draft falls (about every second sequence here)
        rows = case["n_seq"] * (1.5 if case["draft_prob"] else 1.0)
        return {"bytes": rows * vocab * e + case["n_seq"] * (case["max_draft"] * 4 * (2 + 2 * e) + 16), "flops": 3 * rows * vocab}
    n = case["rows"] * vocab
    if case["kind"] == "top":
        return {"bytes": n * e + case["rows"] * (8 * case["k"] + 4), "flops": 4 * n}
    if case["kind"] == "softmax":
        return {"bytes": n * (e + size[case["out"]]), "flops": 4 * n}
    return {"bytes": n * (e + size[case["out"]]) + case["rows"] * (8 * case["k"] + 12), "flops": 6 * n}
