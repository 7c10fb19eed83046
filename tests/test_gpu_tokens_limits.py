"""GPU: the token operators where a value has no bound or a size has no room: infinite margins of the preference loss,
derivatives that they do not have, sizes beyond 32 bits, long sums.  Against plain 64-bit forms; the tolerances of single values
are those of test_gpu_tokens.py (U half a step of fp32, LOGP the error of a log-probability)."""
import pytest
import torch

from test_gpu_tokens import LOGP, U, gen, ids_of, logp_oracle, owner_of, seq_sum, tk, within  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ infinite margins
# (up to 1024 rows and pairs one block computes the loss, beyond that several)
@pytest.mark.parametrize("T,P", [(64, 8), (1024, 30), (1025, 30), (5000, 1100)])
@pytest.mark.parametrize("e", [0.0, 0.1])
@pytest.mark.parametrize("side", ["preferred", "other", "both", "neither"])
def test_infinite_margins(tk, T, P, e, side):
    """A chosen id whose logit is -inf has log-probability -inf.  In the sequence that is not preferred it makes the margin +inf:
    the pair's loss is 0 without label smoothing and inf with it; in the preferred one -inf, and the loss is inf.  The
    gradient is finite: its factor beta (sigmoid(z) - 1 + e) is."""
    g = gen(T + P)
    beta = 0.3
    ptr = torch.linspace(0, T, 2 * P + 1, device="cuda").long().int()
    x, ids = torch.randn(T, 119, device="cuda", generator=g), ids_of(T, 119, g)
    owner = owner_of(ptr, T)
    mask = lambda s: (owner == s).nonzero()[0, 0]   # noqa: E731  (the sequence's first row)
    if side in ("other", "both"):
        t = mask(P + 3)
        x[t, ids[t]] = float("-inf")
    if side in ("preferred", "both"):
        t = mask(5)
        x[t, ids[t]] = float("-inf")
    lp, p, _ = logp_oracle(x, ids)
    r = seq_sum(lp, owner, 2 * P)
    z = beta * (r[:P] - r[P:])
    sp = torch.nn.functional.softplus
    each = (1 - e) * sp(-z) + (e * sp(z) if e else 0.0)
    want = each.mean()
    assert want.isinf() == (side in ("preferred", "both") or (side == "other" and e > 0)) and not want.isnan()
    n = torch.bincount(owner, minlength=2 * P).double()
    slack = beta * ((n + 1) * (LOGP + U)).sum() / P
    got = tk.preference_loss_and_grad(x, ids, ptr, beta=beta, label_smoothing=e)
    within(got.loss, want, slack if want.isfinite() else 0.0, "loss")
    assert got.d_logits.isfinite().all()
    coef = beta * (torch.sigmoid(z) - 1 + e) / P
    if side in ("other", "both"):
        assert got.margin[3] == float("inf") and coef[3] == beta * e / P
        if e == 0:
            assert not got.d_logits[owner == 3].any() and not got.d_logits[owner == P + 3].any()
    if side in ("preferred", "both"):
        assert got.margin[5] == float("-inf")
        rows = owner == 5
        d = -p[rows]
        d[torch.arange(int(rows.sum()), device="cuda"), ids[rows]] += 1
        d *= coef[5]
        within(got.d_logits[rows], d, 3 * LOGP * beta / P * (p[rows] + 1e-3) + 4 * U * d.abs(), "d_logits")
    leaf = x.clone().requires_grad_()
    loss = tk.preference_loss(leaf, ids, ptr, beta=beta, label_smoothing=e).loss
    assert torch.equal(loss, got.loss)
    loss.backward()
    within(leaf.grad, got.d_logits.double(), 4 * U * got.d_logits.abs().double(), "autograd")


def test_nan_margin_is_the_loss(tk):
    """NaN in a sequence, and -inf on both sides of a pair, leave the pair's loss undefined: NaN."""
    x, ids = torch.zeros(8, 9, device="cuda"), torch.zeros(8, dtype=torch.int64, device="cuda")
    ptr = torch.tensor([0, 2, 4, 6, 8], device="cuda")
    for bad in ("nan", "inf - inf"):
        y = x.clone()
        if bad == "nan":
            y[1, 5] = float("nan")
        else:
            y[1, 0] = y[5, 0] = float("-inf")
        for e in (0.0, 0.2):
            assert tk.preference_loss(y, ids, ptr, label_smoothing=e).loss.isnan()


# ------------------------------------------------------------------------------------------------ other derivatives
def test_no_tangent_is_lost(tk):
    """Forward-mode derivatives are refused in every input that has values, and so are torch.func's transforms."""
    import torch.autograd.forward_ad as fw
    g = gen(31)
    x, table = torch.randn(12, 9, device="cuda", generator=g), torch.randn(9, 6, device="cuda", generator=g)
    ids, ptr = ids_of(12, 9, g), torch.tensor([0, 3, 6, 9, 12], device="cuda")
    lp, adv, up = torch.randn(12, device="cuda"), torch.randn(4, device="cuda"), torch.randn(12, 6, device="cuda")
    calls = [(x, lambda y: tk.token_logprobs(y, ids)), (table, lambda y: tk.embed_tokens(ids, y)), (up, lambda y: tk.embed_tokens_grad(y, ids, 9)),
             (torch.zeros(9, 6, device="cuda"), lambda y: tk.embed_tokens_grad(up, ids, 9, out=y))]
    for f in (tk.preference_loss, tk.preference_loss_and_grad):
        calls += [(x, lambda y, f=f: f(y, ids, ptr, lp)), (lp, lambda y, f=f: f(x, ids, ptr, y))]
    for f in (tk.policy_loss, tk.policy_loss_and_grad):
        calls += [(x, lambda y, f=f: f(y, ids, ptr, adv, lp, lp)), (adv, lambda y, f=f: f(x, ids, ptr, y, lp, lp)),
                  (lp, lambda y, f=f: f(x, ids, ptr, adv, y, lp)), (lp, lambda y, f=f: f(x, ids, ptr, adv, lp, y))]
    for i, (t, f) in enumerate(calls):
        with fw.dual_level():
            f(t.clone())                            # no tangent: as ever
            for leaf in (t.clone(), t.clone().requires_grad_()):
                with pytest.raises(NotImplementedError):
                    print(i, f(fw.make_dual(leaf, torch.ones_like(t))))
        with pytest.raises(NotImplementedError, match="tangent"):
            torch.func.jvp(lambda y: f(y) if torch.is_tensor(f(y)) else f(y).loss, (t,), (t,))
        f(t.clone())
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda y: tk.token_logprobs(y, ids))(x.expand(3, 12, 9))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda y: tk.token_logprobs(y, ids).sum())(x)


# ------------------------------------------------------------------------------------------------ sizes beyond 32 bits
@pytest.mark.parametrize("size", [1 << 31, (1 << 32) + 5])
def test_sizes_that_do_not_fit(tk, size):
    """Sizes that the library holds in 32 bits are refused beyond them (2^32 + 5 would arrive as 5).  The tensors are one element
    each, expanded."""
    one, ids = torch.ones(1, 1, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    wide, ptr = one.expand(1, size), torch.zeros(1, dtype=torch.int32, device="cuda").expand(size | 1)
    adv = torch.ones(1, device="cuda")
    for call in (lambda: tk.token_logprobs(wide, ids), lambda: tk.embed_tokens(ids, wide), lambda: tk.embed_tokens_grad(wide, ids, 3),
                 lambda: tk.policy_loss(wide, ids, None, adv), lambda: tk.preference_loss(wide, ids, ptr[:3]),
                 lambda: tk.preference_loss(one, ids, ptr), lambda: tk.policy_loss(one, ids, ptr, adv.expand(size)),
                 lambda: tk.policy_loss_and_grad(one, ids, ptr, adv, advantage_per="token")):
        with pytest.raises(ValueError):
            call()


def test_offsets_beyond_every_position(tk):
    """First positions before 0 and behind the last position, also such as 32 bits do not hold: the sequences reach as far as the
    positions do."""
    g = gen(33)
    T = 1500
    x, ids, adv = torch.randn(T, 9, device="cuda", generator=g), ids_of(T, 9, g, 0.1), torch.randn(2, device="cuda", generator=g)
    of = lambda *v: torch.tensor(v, device="cuda")   # noqa: E731
    for n in (T, 50):                                # (several chunks, and one block)
        want_p = tk.policy_loss_and_grad(x[:n], ids[:n], of(0, 20, n).int(), adv, kl_coef=0.0, aggregate="sequence")
        want_q = tk.preference_loss_and_grad(x[:n], ids[:n], of(0, 20, n).int())
        for ptr in (of(0, 20, n), of(-5, 20, n + 9), of(0, 20, 1 << 31), of(0, 20, (1 << 32) + 3), of(-(1 << 31) - 1, 20, 1 << 40),
                    of(-(1 << 62), 20, (1 << 62) + 25), of(-(1 << 31), 20, (1 << 31) - 1).int()):
            for got, want in ((tk.policy_loss_and_grad(x[:n], ids[:n], ptr, adv, kl_coef=0.0, aggregate="sequence"), want_p),
                              (tk.preference_loss_and_grad(x[:n], ids[:n], ptr), want_q)):
                assert all(torch.equal(a, b) for a, b in zip(got, want)), ptr.tolist()


def test_denominators_at_the_ends(tk):
    """The smallest and largest normal numbers of fp32 divide; what rounds to 0 there is refused (0 asks for the count)."""
    g = gen(34)
    x, ids, ptr = torch.randn(4, 9, device="cuda", generator=g), ids_of(4, 9, g), torch.tensor([0, 2, 4], device="cuda")
    adv = torch.ones(2, device="cuda")
    for f in (lambda d: tk.preference_loss(x, ids, ptr, denominator=d), lambda d: tk.policy_loss(x, ids, ptr, adv, denominator=d)):
        one = f(1.0).loss.double()
        for d in (2.0 ** -126, 2.0 ** -100, 2.0 ** 100, 2.0 ** 127):
            within(f(d).loss, (one / d).float().double(), 2 * U * (one / d).abs(), d)
        for d in (0.0, 1e-50, 1e-40, -1.0, 3.5e38, float("nan"), float("inf")):
            with pytest.raises(ValueError, match="denominator"):
                f(d)


# ------------------------------------------------------------------------------------------------ long sums
@pytest.mark.parametrize("T,V,D", [(65536, 119, 2048), (8192, 119, 16448), (24576, 20, 16448), (16384, 64, 16384), (70000, 300, 1000)])
def test_long_sums_into_small_tables(tk, T, V, D):
    """Every position has one token and the value 1 + 2^-14.  Sums of up to 1023 such values are exact in fp32; from 1024 on an
    addition of one more loses its 2^-14, always to the same side, so that a running sum of 2048 is short by 3e-5.  Parts of
    1024 at most cost one such step (u relative); they are joined four to a block, and the blocks' parts by 8 waves in turn."""
    d = torch.full((T, D), 1 + 2.0 ** -14, device="cuda")
    ids = torch.full((T,), V - 1, device="cuda")
    ids[::97] = -1
    n = int((ids >= 0).sum())
    got = tk.embed_tokens_grad(d, ids, V)
    adds = 1 + 4 + (T / 4096 + 8) + 8
    within(got[V - 1], torch.full((D,), n * (1 + 2.0 ** -14), dtype=torch.float64, device="cuda"), adds * U * n, "sum")
    assert not got[:V - 1].any()
    assert torch.equal(got, tk.embed_tokens_grad(d, ids, V))


@pytest.mark.parametrize("dtype,low", [(torch.bfloat16, -16.75), (torch.float16, -16.640625)])
@pytest.mark.parametrize("V", [1024, 1536, 2048, 6144, 8192, 16384, 24576, 32768, 49152, 98304, 131072])
def test_sums_that_start_with_the_largest(tk, dtype, low, V):
    """One logit 0, all others ``low``: their exponentials are just below half a step of 1 (0.892 and 0.995 u), and each that is
    added to the largest one alone is lost.  The sum is held to the 64 additions a lane and 40 of the tree, one u each, that a
    row's tolerance counts; the other lanes' sums are exact to a few u of 1e-2 at most."""
    x = torch.full((5, V), low, dtype=dtype, device="cuda")
    x[:, 0] = 0
    ids = torch.zeros(5, dtype=torch.int64, device="cuda")
    want = -torch.log1p((V - 1) * torch.tensor(low, dtype=torch.float64, device="cuda").exp()).expand(5)
    within(tk.token_logprobs(x, ids), want, 104 * U, "log-probabilities")
    for T in (1, 5):
        r = tk.policy_loss_and_grad(x[:T], ids[:T], None, torch.ones(1, device="cuda"), kl_coef=0.0)
        within(r.logp, want[:T], 104 * U, "policy")


def test_more_sequences_than_one_launch_holds(tk):
    """A wave for each of 68 million sequences would be more than the 2^32 threads of a launch.  Nearly all are empty."""
    g = gen(36)
    T, S = 1500, 68_000_000
    x, ids = torch.randn(T, 9, device="cuda", generator=g), ids_of(T, 9, g, 0.1)
    few = torch.tensor([0, 400, 1100, T], device="cuda", dtype=torch.int32)
    ptr = torch.zeros(S + 1, dtype=torch.int32, device="cuda")
    ptr[S // 2:], ptr[-2:], ptr[-1:] = 400, 1100, T        # the last three are not empty
    ptr[S - 2] = 400
    adv = torch.zeros(S, device="cuda")
    adv[S // 2 - 1], adv[-2:] = 0.3, torch.tensor([-1.2, 0.7], device="cuda")
    got = tk.policy_loss_and_grad(x, ids, ptr, adv, kl_coef=0.0, aggregate="sequence", denominator=3)
    want = tk.policy_loss_and_grad(x, ids, few, torch.tensor([0.3, -1.2, 0.7], device="cuda"), kl_coef=0.0, aggregate="sequence")
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and bool(got.d_logits.any())
