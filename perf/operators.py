"""Operators of a serving step around the lm_head and the sampler, measured on
device-resident buffers the way a decode loop calls them.

Three operators:
  verify      Sampler.verify_drafts_device: drafted tokens against whole rows
              of the target's logits (or probabilities), from given uniforms
  candidates  Sampler.verify_candidates_device: the same against the candidate
              lists that Sampler.sample_device writes (top-k / top-p truncated)
  lora        Sampler.lora_device: the low-rank adapter of each row's request
              beside a projection's result; Sampler.gemv_lora_device with the
              shared projection in the same call

The ragged layout of verify and candidates: sequence b has its drafts at
off[b] .. off[b + 1], its target rows (one more than drafts), uniforms and
output tokens at off[b] + b ..., its draft rows at off[b] ....

Every plain form is written in torch's elementary operations.  Draws compare a
uniform with running sums over a whole vocabulary, whose steps lie near 1e-7 of
the total, so distributions are formed in binary64; adapters in binary32.
"""
import torch

own = False

V = 151936                    # the workloads' vocabulary
NONE = -1                     # behind a sequence's last token
# what a drawn case may cost at most, from the largest listed ones: logits of
# target and draft rows; candidate entries; results; adapter elements
MAX_LOGITS = 17 * 64 * V
MAX_ENTRIES = 5 * 32 * 1024
MAX_RESULTS = 2048 * 4096
MAX_ADAPTER = 32 * 16 * V
NOISE = 1.2                   # a draft model's logits are off the target's by this (rms)
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}


def listed():
    return [
        # one sequence with prompt-lookup drafts (no draft model): the smallest call
        dict(name="verify-lookup-1", op="verify", seqs=1, drafts=3, ragged=False, vocab=V,
             target="logits", draft="none", pad=0),
        # a small batch behind a draft model
        dict(name="verify-16", op="verify", seqs=16, drafts=4, ragged=False, vocab=V,
             target="logits", draft="logits", pad=0),
        # drafts of different lengths, the draft's probabilities kept, a row
        # length that is no multiple of 4, an odd vocabulary
        dict(name="verify-ragged-50", op="verify", seqs=50, drafts=7, ragged=True, vocab=40007,
             target="logits", draft="probs", pad=2),
        # a server that keeps probabilities on both sides
        dict(name="verify-probs-32", op="verify", seqs=32, drafts=5, ragged=True, vocab=V,
             target="probs", draft="probs", pad=0),
        # a large batch with long drafts: the largest
        dict(name="verify-64", op="verify", seqs=64, drafts=8, ragged=False, vocab=V,
             target="logits", draft="logits", pad=0),
        # a few sequences sampled with top-k 40
        dict(name="candidates-4", op="candidates", seqs=4, drafts=3, ragged=False, vocab=V, k=40,
             draft=True),
        # the benchmark's batch, top-k 20, ragged
        dict(name="candidates-256", op="candidates", seqs=256, drafts=4, ragged=True, vocab=V, k=20,
             draft=True),
        # the longest lists of the select kernels
        dict(name="candidates-k1024", op="candidates", seqs=32, drafts=4, ragged=False, vocab=V,
             k=1024, draft=True),
        # one request's adapter on the lm_head
        dict(name="lora-1", op="lora", m=1, hidden=2048, out=V, rank=16, type="bf16", count=8,
             used=1, ragged=False, project=False),
        # a decode batch, an adapter for every request
        dict(name="lora-32", op="lora", m=32, hidden=2048, out=V, rank=16, type="bf16", count=32,
             used=32, ragged=False, project=False),
        # odd sizes, ranks of their own, requests without an adapter, beside
        # the projection itself
        dict(name="project-lora-7", op="lora", m=7, hidden=1024, out=32007, rank=24, type="f16",
             count=6, used=4, ragged=True, project=True),
        # a few prompts of different lengths through an inner projection
        dict(name="lora-prompts-2048", op="lora", m=2048, hidden=4096, out=4096, rank=64,
             type="bf16", count=8, used=6, ragged=False, project=False),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["verify", "verify", "candidates", "lora", "lora"])
    if op == "verify":
        seqs, drafts = _log(rng, 1, 64), rng.randint(1, 8)
        vocab = V if rng.random() < 0.3 else _log(rng, 1000, 262144)
        vocab = min(vocab, MAX_LOGITS // (seqs * (2 * drafts + 1)))
        return dict(op=op, seqs=seqs, drafts=drafts, ragged=rng.random() < 0.5, vocab=vocab,
                    target=rng.choice(["logits", "logits", "probs"]),
                    draft=rng.choice(["logits", "probs", "none"]), pad=rng.choice([0, 0, 1, 4, 9]))
    if op == "candidates":
        seqs, drafts, k = _log(rng, 1, 256), rng.randint(1, 8), _log(rng, 2, 1024)
        seqs = min(seqs, max(1, MAX_ENTRIES // ((drafts + 1) * k)))
        return dict(op=op, seqs=seqs, drafts=drafts, ragged=rng.random() < 0.5,
                    vocab=_log(rng, 32000, 262144), k=k, draft=rng.random() < 0.8)
    out = _log(rng, 256, V)
    m = _log(rng, 1, min(2048, MAX_RESULTS // out))
    kind, rank = rng.choice(["bf16", "bf16", "f16", "f32"]), _log(rng, 1, 128)
    size = 2 if kind == "f32" else 1
    count = _log(rng, 1, max(1, min(32, MAX_ADAPTER // (out * rank * size))))
    project = m <= 16 and out <= 33000 and rng.random() < 0.3
    hidden = 64 * rng.randint(1, 64) if project else _log(rng, 64, 4096)
    return dict(op=op, m=m, hidden=hidden, out=out, rank=rank, type=kind, count=count,
                used=min(m, rng.randint(1, count)), ragged=rng.random() < 0.5, project=project)


# ---- inputs ---------------------------------------------------------------

def _lengths(case):
    """Drafts of each sequence, a function of the case alone."""
    n, d = case["seqs"], case["drafts"]
    if not case["ragged"] or n == 1:
        return [d] * n
    return [(b * 5 + b // 3 + 2) % (d + 1) for b in range(n - 1)] + [d]


def _layout(case):
    """off and, for every draft, its target row."""
    lens = torch.tensor(_lengths(case), device="cuda")
    off = torch.zeros(case["seqs"] + 1, dtype=torch.int64, device="cuda")
    off[1:] = lens.cumsum(0)
    return off


def _logits(rows, vocab, g):
    x = torch.empty(rows, vocab, device="cuda").normal_(0.0, 2.5, generator=g)
    top = torch.randint(0, vocab, (rows, 8), device="cuda", generator=g)
    return x.scatter_add_(1, top, torch.full((rows, 8), 12.0, device="cuda"))


def _drawn(p, g):
    """A draw of each row of probabilities."""
    e = torch.empty_like(p).exponential_(generator=g).clamp_(min=1e-30)
    return (p / e).argmax(-1)


def _padded(rows, pad):
    """Rows a little longer than the vocabulary."""
    if not pad:
        return rows
    return torch.cat([rows, torch.zeros(rows.shape[0], pad, device="cuda")], 1).contiguous()


def _verify_inputs(case, g):
    off = _layout(case)
    seqs, vocab, total = case["seqs"], case["vocab"], sum(_lengths(case))
    temps = torch.rand(seqs, device="cuda", dtype=torch.float64, generator=g) * 0.9 + 0.3
    temps[torch.arange(seqs, device="cuda") % 8 == 5] = 0.0      # some decode greedily
    lens = off[1:] - off[:-1]
    seq_d = torch.repeat_interleave(torch.arange(seqs, device="cuda"), lens, output_size=total)
    at = torch.arange(total, device="cuda") + seq_d               # a draft's target row
    seq_t = torch.repeat_interleave(torch.arange(seqs, device="cuda"), lens + 1,
                                    output_size=total + seqs)
    target = _logits(total + seqs, vocab, g)
    draft = target[at]
    if case["draft"] != "none":
        draft = draft + torch.empty_like(draft).normal_(0.0, NOISE, generator=g)
    warm = temps.clamp(min=0.3).float()
    q = torch.softmax(draft / warm[seq_d, None], -1)
    ids = _drawn(q, g)
    s = dict(temps=temps, off=off, ids=ids.to(torch.int32),
             u=torch.rand(total + seqs, device="cuda", dtype=torch.float64, generator=g))
    if case["target"] == "probs":
        target = torch.softmax(target / warm[seq_t, None], -1)
    s["target"] = _padded(target, case["pad"])
    if case["draft"] != "none":
        s["draft"] = _padded(q if case["draft"] == "probs" else draft, case["pad"])
        # the draft model samples at the target's temperature, never greedily
        s["draft_temps"] = temps.clamp(min=0.3)
    return s


def _lists(logits, ids, k):
    """Sorted candidates of each row (ids, probabilities, kept prefix at top-p
    0.95), as the sampler writes them."""
    v, j = logits.topk(k, -1)
    p = torch.softmax(v.double(), -1).float()
    kept = (p.double().cumsum(-1) < 0.95).sum(-1) + 1
    return ids.gather(1, j), p, kept.clamp(max=k).to(torch.int32)


def _candidate_inputs(case, g):
    off = _layout(case)
    seqs, k, total = case["seqs"], case["k"], sum(_lengths(case))
    lens = off[1:] - off[:-1]
    seq_d = torch.repeat_interleave(torch.arange(seqs, device="cuda"), lens, output_size=total)
    at = torch.arange(total, device="cuda") + seq_d
    pool = 2 * k + 8                                              # ids near the top of a row
    start = torch.randint(0, case["vocab"], (total + seqs, 1), device="cuda", generator=g)
    ids = ((start + 7 * torch.arange(pool, device="cuda")) % case["vocab"]).to(torch.int32)
    x = torch.empty(total + seqs, pool, device="cuda").normal_(0.0, 2.5, generator=g)
    t = _lists(x, ids, k)
    near = x[at] + torch.empty(total, pool, device="cuda").normal_(0.0, NOISE, generator=g)
    d = _lists(near, ids[at], k)
    kept = torch.arange(k, device="cuda") < d[2][:, None]
    pick = _drawn(torch.where(kept, d[1], 0.0), g)
    s = dict(off=off, ids=d[0].gather(1, pick[:, None])[:, 0].contiguous(), t=t,
             u=torch.rand(total + seqs, device="cuda", dtype=torch.float64, generator=g))
    if case["draft"]:
        s["d"] = d
    return s


def _slots(case):
    """The adapter of each row: `used` of them, in runs for prompts (more rows
    than adapters by far), in turn for a decode batch; ragged: every fourth
    row of a batch has none."""
    m, used, count = case["m"], case["used"], case["count"]
    r = torch.arange(m)
    s = r * used // m if m > 64 else r % used
    s = (s * 5 + 3) % count if count % 5 else (s * 3 + 1) % count if count % 3 else s
    if case["ragged"]:
        s[r % 4 == 3] = -1
    return s.to(torch.int32)


def _ranks(case):
    """The rank of each adapter, at most the stacks'."""
    c = torch.arange(case["count"])
    r = case["rank"]
    return (r - (c * 7) % max(1, r) * (1 if case["ragged"] else 0)).to(torch.int32)


def _lora_inputs(case, g):
    m, K, N, r, n = case["m"], case["hidden"], case["out"], case["rank"], case["count"]
    dt = DTYPES[case["type"]]
    big = torch.rand(K, device="cuda", generator=g) < 0.01
    x = torch.empty(m, K, device="cuda").normal_(0.0, 1.0, generator=g)
    s = dict(x=torch.where(big, x * 10.0, x).contiguous(),
             a=torch.empty(n, r, K, device="cuda", dtype=dt).normal_(0.0, K ** -0.5, generator=g),
             b=torch.empty(n, N, r, device="cuda", dtype=dt).normal_(0.0, 0.5, generator=g),
             scales=torch.rand(n, device="cuda", generator=g) + 0.5,
             ranks=_ranks(case).cuda(), slots=_slots(case).cuda())
    if case["project"]:
        s["w"] = torch.empty(N, K, device="cuda").normal_(0.0, 1.8 / K ** 0.5, generator=g)
    else:
        s["base"] = torch.empty(m, N, device="cuda").normal_(0.0, 2.5, generator=g)
    return s


def _inputs(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed * 7919 + case.get("vocab", case.get("out")))
    make = dict(verify=_verify_inputs, candidates=_candidate_inputs, lora=_lora_inputs)
    return make[case["op"]](case, g)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    if case["op"] == "lora":
        s["y"] = torch.empty(case["m"], case["out"], device="cuda")
    else:
        total = sum(_lengths(case))
        s["total"] = total
        s["tokens"] = torch.empty(total + case["seqs"], dtype=torch.int32, device="cuda")
        s["counts"] = torch.empty(case["seqs"], dtype=torch.int32, device="cuda")
        s["accept"] = torch.empty(total, device="cuda")
    return s


# ---- the plain forms --------------------------------------------------------

def _distribution(rows, kind, temps):
    """Binary64 probabilities of rows of logits at a temperature each (<= 0:
    all on the first maximum), or of rows of probabilities."""
    if kind == "probs":
        return rows.double()
    x = rows.double()
    top, first = x.max(-1, keepdim=True)
    greedy = (temps <= 0)[:, None]
    w = torch.exp((x - top) / torch.where(greedy, 1.0, temps[:, None]))
    w /= w.sum(-1, keepdim=True)
    only = torch.arange(x.shape[1], device=x.device) == first
    return torch.where(greedy, only.double(), w)


def _outcome(s, px, qx):
    """Accepted drafts of each sequence and the judged acceptance
    probabilities, from the drafts' probabilities on both sides."""
    off, u, seqs = s["off"], s["u"], s["case"]["seqs"]
    lens = off[1:] - off[:-1]
    d = torch.arange(s["total"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), lens, output_size=s["total"])
    ok = u[d + seq] * qx < px
    pos = d - off[seq]
    big = s["case"]["drafts"] + 1
    first = torch.full((seqs,), big, dtype=torch.int64, device="cuda")
    first = first.scatter_reduce(0, seq, torch.where(ok, big, pos), "amin")
    n = torch.minimum(first, lens)
    ratio = torch.where(px >= qx, 1.0, px / torch.where(qx > 0, qx, 1.0))
    accept = torch.where(pos <= n[seq], ratio, 0.0).float()
    return lens, seq, pos, n, accept


def _emit(s, lens, seq, pos, n, accept, final):
    """Tokens of the ragged layout: accepted drafts, the final token, -1s."""
    seqs, total = s["case"]["seqs"], s["total"]
    b = torch.arange(seqs, device="cuda")
    tokens = torch.full((total + seqs,), NONE, dtype=torch.int32, device="cuda")
    at = torch.arange(total, device="cuda") + seq
    tokens[at] = torch.where(pos < n[seq], s["ids"], NONE)
    tokens[s["off"][:-1] + b + n] = final.to(torch.int32)
    return dict(tokens=tokens, counts=(n + 1).to(torch.int32), accept=accept)


def _rest(p, q, certain, x, take):
    """What a final token is drawn from: p where every draft was accepted
    (`take`), else p beyond q (or p without the certain draft x), else p."""
    if certain:
        r = p.scatter(1, x[:, None], 0.0)
    else:
        r = (p - q).clamp(min=0.0)
    r = torch.where(take[:, None], p, r)
    return torch.where(r.sum(-1, keepdim=True) > 0, r, p)


def _pick(r, u):
    """The first position whose running sum is above u times the whole."""
    c = r.cumsum(-1)
    return torch.searchsorted(c, (u * c[:, -1])[:, None], right=True)[:, 0].clamp(max=r.shape[1] - 1)


def _verify(s):
    c = s["case"]
    vocab, seqs, off = c["vocab"], c["seqs"], s["off"]
    lens = off[1:] - off[:-1]
    b = torch.arange(seqs, device="cuda")
    seq_t = torch.repeat_interleave(b, lens + 1, output_size=s["total"] + seqs)
    seq_d = torch.repeat_interleave(b, lens, output_size=s["total"])
    at = torch.arange(s["total"], device="cuda") + seq_d
    x = s["ids"].long()
    p = _distribution(s["target"][:, :vocab], c["target"], s["temps"][seq_t])
    px = p[at, x]
    certain = c["draft"] == "none"
    if certain:
        qx = torch.ones_like(px)
    else:
        q = _distribution(s["draft"][:, :vocab], c["draft"], s["draft_temps"][seq_d])
        qx = q.gather(1, x[:, None])[:, 0]
    lens, seq, pos, n, accept = _outcome(s, px, qx)
    start = off[:-1] + b
    last = (off[:-1] + n).clamp(max=max(0, s["total"] - 1))
    final = _rest(p[start + n], None if certain else q[last], certain, x[last], n == lens)
    return _emit(s, lens, seq, pos, n, accept, _pick(final, s["u"][start + lens]))


def _candidates(s):
    c = s["case"]
    k, seqs, off = c["k"], c["seqs"], s["off"]
    b = torch.arange(seqs, device="cuda")
    seq_d = torch.repeat_interleave(b, off[1:] - off[:-1], output_size=s["total"])
    at = torch.arange(s["total"], device="cuda") + seq_d
    x = s["ids"][:, None]
    inside = torch.arange(k, device="cuda")

    def weights(lists):
        w = torch.where(inside < lists[2][:, None], lists[1], 0.0).double()
        return lists[0], w / w.sum(-1, keepdim=True)

    ids, p = weights(s["t"])
    px = torch.where(ids[at] == x, p[at], 0.0).sum(-1)
    if c["draft"]:
        dids, q = weights(s["d"])
        qx = torch.where(dids == x, q, 0.0).sum(-1)
    else:
        qx = torch.ones_like(px)
    lens, seq, pos, n, accept = _outcome(s, px, qx)
    start = off[:-1] + b
    row, last = start + n, (off[:-1] + n).clamp(max=max(0, s["total"] - 1))
    p, ids = p[row], ids[row]
    if c["draft"]:
        same = ids[:, :, None] == dids[last][:, None, :]
        r = (p - torch.where(same, q[last][:, None, :], 0.0).sum(-1)).clamp(min=0.0)
    else:
        r = torch.where(ids == x[last], 0.0, p)
    r = torch.where((n == lens)[:, None], p, r)
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, p)
    final = ids.gather(1, _pick(r, s["u"][start + lens])[:, None])[:, 0]
    return _emit(s, lens, seq, pos, n, accept, final)


def _lora(s):
    c = s["case"]
    m, r, n = c["m"], c["rank"], c["count"]
    y = s["x"] @ s["w"].t() if c["project"] else s["base"]
    slots = s["slots"].long()
    has = slots >= 0
    slot = slots.clamp(min=0)
    live = torch.arange(r, device="cuda") < s["ranks"][:, None]            # [n, r]
    scale = torch.where(has, s["scales"][slot], 0.0)[:, None]
    if m <= n:                          # the rows' own adapters
        a = torch.where(live[slot][:, :, None], s["a"][slot].float(), 0.0)
        t = (a @ s["x"][:, :, None]) * scale[:, :, None]
        b = torch.where(live[slot][:, None, :], s["b"][slot].float(), 0.0)
        return y + (b @ t)[:, :, 0]
    # more rows than adapters: all adapters side by side, the others' columns 0
    a = torch.where(live[:, :, None], s["a"].float(), 0.0).reshape(n * r, -1)
    t = (s["x"] @ a.t()).reshape(m, n, r) * scale[:, :, None]
    t = torch.where((torch.arange(n, device="cuda") == slot[:, None])[:, :, None], t, 0.0)
    b = torch.where(live[:, None, :], s["b"].float(), 0.0).transpose(1, 2).reshape(n * r, -1)
    return y + t.reshape(m, n * r) @ b


# ---- the framework's operators --------------------------------------------------

_SAMPLER = None


def _call(s):
    """The call's descriptors over the state's buffers, made once as a serving
    loop makes them for the buffers that it keeps."""
    global _SAMPLER
    from hachiue_amd import Sampler
    from hachiue_amd import sampler as hs
    if _SAMPLER is None:
        _SAMPLER = Sampler(0)
    c, st = s["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "lora":
        ad = hs.adapters(GGML[c["type"]], c["count"], c["rank"], c["hidden"], c["out"],
                         s["a"].data_ptr(), s["b"].data_ptr(), s["scales"].data_ptr(),
                         s["ranks"].data_ptr())
        x, y, slots = s["x"].data_ptr(), s["y"].data_ptr(), s["slots"].data_ptr()
        m, K, N = c["m"], c["hidden"], c["out"]
        if c["project"]:
            w = hs.weights(0, N, K, s["w"].data_ptr())
            return _SAMPLER.gemv_lora_device, (x, m, K, w, ad, slots, y, N, st)
        return _SAMPLER.lora_device, (x, m, K, ad, slots, s["base"].data_ptr(), N, y, N, st)
    batch = hs.draft_batch(c["seqs"], c["drafts"], s["total"], s["off"].data_ptr(),
                           s["ids"].data_ptr(), s["u"].data_ptr(), s["tokens"].data_ptr(),
                           s["counts"].data_ptr(), s["accept"].data_ptr())
    if c["op"] == "verify":
        kinds, ld = dict(logits=hs.DIST_LOGITS, probs=hs.DIST_PROBS), c["vocab"] + c["pad"]
        t = hs.distribution(kinds[c["target"]], s["target"].data_ptr(), ld, s["temps"].data_ptr())
        d = None
        if c["draft"] != "none":
            d = hs.distribution(kinds[c["draft"]], s["draft"].data_ptr(), ld,
                                s["draft_temps"].data_ptr())
        return _SAMPLER.verify_drafts_device, (t, d, c["vocab"], batch, None, st)
    t = hs.candidates(c["k"], *(x.data_ptr() for x in s["t"]))
    d = hs.candidates(c["k"], *(x.data_ptr() for x in s["d"])) if c["draft"] else None
    return _SAMPLER.verify_candidates_device, (t, d, batch, None, st)


def run(s):
    op = s["case"]["op"]
    if not own:
        return dict(verify=_verify, candidates=_candidates, lora=_lora)[op](s)
    if "call" not in s:
        s["call"] = _call(s)
    f, args = s["call"]
    f(*args)
    return s["y"] if op == "lora" else {k: s[k] for k in ("tokens", "counts", "accept")}


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    """verify: every row read once (how many of a sequence's rows are needed
    turns out only as they are judged), or, where the rows are probabilities,
    one element of each and the rows that the final token is drawn from.
    candidates: every list once.  lora: hidden states, the adapters in use,
    base (or weights) read once, results written once."""
    if case["op"] == "lora":
        m, K, N = case["m"], case["hidden"], case["out"]
        slots, ranks = _slots(case), _ranks(case)
        size = 4 if case["type"] == "f32" else 2
        live = slots[slots >= 0].long()
        n = int(ranks[live.unique()].sum()) * (K + N) * size + 4 * (m * K + m * N)
        flops = 2 * int(ranks[live].sum()) * (K + N)
        n += 4 * (N * K if case["project"] else m * N)
        flops += 2 * m * N * K if case["project"] else m * N
        return dict(bytes=n, flops=flops)
    lens = _lengths(case)
    seqs, total = case["seqs"], sum(lens)
    small = 4 * total + 8 * (total + seqs) + 8 * (seqs + 1) + 4 * (total + seqs) + 4 * seqs + 4 * total
    if case["op"] == "candidates":
        rows = total + seqs + (total if case["draft"] else 0)
        return dict(bytes=small + rows * (8 * case["k"] + 4), flops=4 * rows * case["k"])
    rows = seqs if case["target"] == "probs" else total + seqs
    if case["draft"] != "none":
        rows += sum(x > 0 for x in lens) if case["draft"] == "probs" else total
    return dict(bytes=small + 4 * rows * case["vocab"], flops=4 * rows * case["vocab"])


# ---- the same in 64 bits ------------------------------------------------------

def _log_p(row, kind, t):
    """Natural logarithms of one row's probabilities."""
    if kind == "probs":
        return row.double().log()
    if t <= 0:
        out = torch.full_like(row, -float("inf"), dtype=torch.float64)
        out[int(row.argmax())] = 0.0
        return out
    z = row.double() / t
    return z - torch.logsumexp(z, 0)


def _walk(case, s, p_row, q_row, prob_at, final_ids):
    """Each sequence by itself, draft after draft."""
    off, u, ids = s["off"].tolist(), s["u"].tolist(), s["ids"].tolist()
    total, seqs = off[-1], case["seqs"]
    tokens = torch.full((total + seqs,), NONE, dtype=torch.int32)
    counts, accept = torch.zeros(seqs, dtype=torch.int32), torch.zeros(total, dtype=torch.float64)
    for b in range(seqs):
        n, at = off[b + 1] - off[b], off[b] + b
        i, q, rejected = 0, None, False
        while i < n and not rejected:
            x, p, q = ids[off[b] + i], p_row(b, at + i), q_row(b, off[b] + i)
            px, qx = prob_at(p, at + i, x), 1.0 if q is None else prob_at(q, off[b] + i, x, True)
            accept[off[b] + i] = 1.0 if px >= qx else px / qx
            rejected = not u[at + i] * qx < px
            if not rejected:
                tokens[at + i] = x
                i += 1
        p = p_row(b, at + i)
        r = final_ids(p, q, at + i, off[b] + i, ids[off[b] + i]) if rejected else p
        if float(r.sum()) <= 0:
            r = p
        c = torch.cumsum(r, 0)
        j = min(int((c <= u[at + n] * float(c[-1])).sum()), r.numel() - 1)
        tokens[at + i] = j if case["op"] == "verify" else int(s["t"][0][at + i][j])
        counts[b] = i + 1
    return dict(tokens=tokens.cuda(), counts=counts.cuda(), accept=accept.cuda())


def _exact_verify(case, s):
    vocab, temps = case["vocab"], s["temps"].tolist()

    def p_row(b, row):
        return _log_p(s["target"][row, :vocab], case["target"], temps[b]).exp()

    def q_row(b, row):
        if case["draft"] == "none":
            return None
        return _log_p(s["draft"][row, :vocab], case["draft"], max(temps[b], 0.3)).exp()

    def rest(p, q, row, drow, x):
        r = p.clone()
        if q is None:
            r[x] = 0.0
            return r
        return torch.maximum(r - q, torch.zeros_like(r))

    return _walk(case, s, p_row, q_row, lambda p, row, x, d=False: float(p[x]), rest)


def _exact_candidates(case, s):
    def row_of(lists, row):
        p = lists[1][row].double()
        p[int(lists[2][row]):] = 0.0
        return p / p.sum()

    def prob_at(p, row, x, d=False):
        return float(p[(s["d"] if d else s["t"])[0][row] == x].sum())

    def rest(p, q, row, drow, x):
        ids = s["t"][0][row].tolist()
        if q is None:
            drop = {x: 2.0}
        else:
            drop = dict(zip(s["d"][0][drow].tolist(), q.tolist()))
        return torch.tensor([max(a - drop.get(i, 0.0), 0.0) for i, a in zip(ids, p.tolist())],
                            dtype=torch.float64)

    def q_row(b, row):
        return row_of(s["d"], row).cpu() if case["draft"] else None

    s = {k: v.cpu() if torch.is_tensor(v) else tuple(x.cpu() for x in v) for k, v in s.items()}
    return _walk(case, s, lambda b, row: row_of(s["t"], row), q_row, prob_at, rest)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "verify":
        return _exact_verify(case, s)
    if case["op"] == "candidates":
        return _exact_candidates(case, s)
    x = s["x"].double()
    y = x @ s["w"].double().t() if case["project"] else s["base"].double()
    slots = s["slots"].tolist()
    for slot in sorted(set(slots) - {-1}):
        rows = torch.tensor([i for i, v in enumerate(slots) if v == slot], device="cuda")
        r = int(s["ranks"][slot])
        t = x[rows] @ s["a"][slot, :r].double().t()
        y[rows] += float(s["scales"][slot]) * (t @ s["b"][slot, :, :r].double().t())
    return y
