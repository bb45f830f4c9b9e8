"""Host-side behaviour of the losses over vocabulary logits: every bad argument is an
error before anything is launched, and no operator runs on CPU tensors."""
import pytest
import torch

from lema_b200 import _native as N
from lema_b200 import ops

FAKE = 4096          # a non-null, aligned address that is never dereferenced
ROWS = (FAKE, 0, 2, 3, 300, 100, 100)


def logprobs(rows=ROWS, targets=FAKE, tau=1.0, logps=FAKE):
    return N.lib().lema_token_logprobs(*rows, targets, -100, tau, logps, None, None)


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    logprobs((None, 0, 0, 3, 300, 100, 100))     # a call that succeeds clears the message
    assert N.last_error() == ""


def test_rows():
    assert logprobs((None, 0, 0, 3, 300, 100, 100)) == N.LEMA_OK       # no rows: nothing to do
    assert logprobs((None, 0, 2, 0, 300, 100, 100)) == N.LEMA_OK
    for rows in ((None, 0, 2, 3, 300, 100, 100), (FAKE, 0, -1, 3, 300, 100, 100),
                 (FAKE, 0, 2, -3, 300, 100, 100), (FAKE, 0, 2, 3, -1, 100, 100),
                 (FAKE, 0, 2, 3, 300, -1, 100), (FAKE, 0, 2, 3, 300, 100, 0),
                 (FAKE, 0, 2, 3, 300, 100, (1 << 30) + 1)):
        assert logprobs(rows) == N.LEMA_ERR_INVALID_ARGUMENT, rows
    assert logprobs((FAKE, 0, 1 << 20, 1 << 20, 1, 1, 1)) == N.LEMA_ERR_UNSUPPORTED
    assert logprobs(targets=None) == N.LEMA_ERR_INVALID_ARGUMENT
    assert logprobs(logps=None) == N.LEMA_ERR_INVALID_ARGUMENT
    for tau in (0.0, -1.0, float("nan"), float("inf"), 1e-7, 1e7):
        assert logprobs(tau=tau) == N.LEMA_ERR_INVALID_ARGUMENT
        assert "temperature" in N.last_error()


def test_workspace_bytes():
    size = N.lib().lema_loss_workspace_bytes
    assert size(-1, 4) == -1 and size(4, -1) == -1 and size(1 << 20, 1 << 20) == -1
    assert 0 < size(0, 0) <= size(2, 3) <= size(8, 512)


def preference(n0=2, ws=FAKE, n=1 << 20, beta=0.1, e=0.0, out=(None, 0, 0), loss=FAKE):
    return N.lib().lema_preference_loss(FAKE, 0, n0, 3, 300, 100, 100, FAKE, -100, None, beta, e,
                                        1.0, ws, n, FAKE, FAKE, FAKE, loss, FAKE, *out, None)


def policy(ws=FAKE, n=1 << 20, clip=(0.2, 0.2), kl=0.0, adv=FAKE, out=(None, 0, 0)):
    return N.lib().lema_policy_loss(FAKE, 0, 2, 3, 300, 100, 100, FAKE, -100, 1.0, None, adv, 3, 1,
                                    None, *clip, kl, 0, 1.0, ws, n, FAKE, None, None, FAKE, FAKE,
                                    *out, None)


def distill(K=3, ids=FAKE, ws=FAKE, n=1 << 20, out=(None, 0, 0)):
    return N.lib().lema_distill_loss(FAKE, 0, 2, 3, 300, 100, 100, ids, 0, FAKE, 1, K, None, 1.0,
                                     1.0, None, ws, n, FAKE, *out, None)


def test_losses_refuse():
    bad = N.LEMA_ERR_INVALID_ARGUMENT
    need = N.lib().lema_loss_workspace_bytes(2, 3)
    for f in (preference, policy, distill):
        assert f(ws=None) == bad and "workspace" in N.last_error()
        assert f(ws=FAKE + 4) == bad
        assert f(n=need - 1) == bad
        assert f(out=(FAKE, 300, 99)) == bad and "overlap" in N.last_error()
        assert f(out=(FAKE, 299, 100)) == bad
        assert f(out=(FAKE, -300, 100)) == bad
    assert preference(n0=3) == bad and preference(n0=0) == bad
    for kw in ({"beta": 0.0}, {"beta": -1.0}, {"beta": float("inf")}, {"e": 0.5}, {"e": -0.1},
               {"e": float("nan")}, {"loss": None}):
        assert preference(**kw) == bad, kw
    for kw in ({"clip": (1.1, 0.2)}, {"clip": (-0.1, 0.2)}, {"clip": (0.2, float("nan"))},
               {"kl": -0.5}, {"kl": float("inf")}, {"adv": None}):
        assert policy(**kw) == bad, kw
    assert distill(K=0) == N.LEMA_ERR_UNSUPPORTED and distill(K=1025) == N.LEMA_ERR_UNSUPPORTED
    assert distill(ids=None) == bad


@pytest.mark.parametrize("name", ["token_logprobs", "preference_loss", "preference_loss_grad",
                                  "policy_loss", "policy_loss_grad", "distill_loss",
                                  "distill_loss_grad"])
def test_no_cpu_fallback(name):
    x = torch.zeros(2, 3, 8, dtype=torch.bfloat16)
    t = torch.zeros(2, 3, dtype=torch.int64)
    ids = torch.zeros(2, 3, 4, dtype=torch.int64)
    args = {"token_logprobs": (t,), "preference_loss": (t,), "policy_loss": (t, None, torch.ones(2)),
            "distill_loss": (ids, ids.float())}[name.replace("_grad", "")]
    for v in (x, x.clone().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            getattr(ops, name)(v, *args)


def test_rows_that_overlap_are_found():
    base = torch.zeros(4, 6, 8)
    assert ops._rows_disjoint(base) and ops._rows_disjoint(base.transpose(0, 1))
    assert ops._rows_disjoint(base[:, ::2, :5]) and ops._rows_disjoint(base[:0])
    assert not ops._rows_disjoint(base[:1].expand(4, 6, 8))
    assert not ops._rows_disjoint(base.transpose(1, 2))
    assert not ops._rows_disjoint(base.as_strided((4, 6, 8), (48, 7, 1)))


def test_next_targets():
    from lema_b200.objectives import next_targets
    labels = torch.tensor([[5, 6, -100, 7], [1, 2, 3, 4]])
    assert next_targets(labels).tolist() == [[6, -100, 7, -100], [2, 3, 4, -100]]


def test_adapters_can_be_left_out():
    from lema_b200.modules import LoRALinear
    base = torch.nn.Linear(8, 6, bias=False)
    m = LoRALinear(base, 2, 4.0, dtype=torch.float32)
    torch.nn.init.normal_(m.lora_B)
    x = torch.randn(3, 8)
    assert not torch.equal(m(x), base(x))
    m.enabled = False
    assert torch.equal(m(x), base(x)) and LoRALinear.enabled


def test_cluster_memory_is_used_behind_a_cluster_barrier():
    """Another CTA's shared memory exists once that CTA runs: every kernel that takes an
    address in it (mapa) has waited at a cluster barrier before. Read from the sources, since
    an access too early is undefined."""
    import re
    from lema_b200 import build
    seen = 0
    for path in build.sources():
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for body in text.split("__global__")[1:]:
            remote = body.find("mapa_shared(")
            if remote < 0:
                continue
            seen += 1
            head = body[:remote]
            assert "cluster_sync()" in head or "cluster_wait()" in head, (path.name, body[:80])
    assert seen >= 2


def test_scores_refuse_longer_sequences():
    """Positions behind the trainer's rotary tables would be read past their end."""
    from types import SimpleNamespace
    from lema_b200.trainer import StreamedLoraTrainer
    tr = SimpleNamespace(seq=8)                 # refused before anything else is touched
    for shape in ((2, 9), (2, 0), (8,), (1, 2, 4)):
        with pytest.raises(ValueError, match="ids"):
            StreamedLoraTrainer.token_logprobs(tr, torch.zeros(shape, dtype=torch.int64))
    ids = torch.zeros(2, 8, dtype=torch.int64)
    with pytest.raises(ValueError, match="labels"):
        StreamedLoraTrainer.token_logprobs(tr, ids, ids[:, 1:])


def test_rope_refuses_short_tables():
    q = torch.zeros(12, 32, dtype=torch.bfloat16)
    table, short = torch.zeros(6, 16), torch.zeros(1, 5, 16)
    for cos, sin in ((short, table), (table, short)):
        with pytest.raises(ValueError, match="cos and sin"):
            ops.rope(q, q, cos, sin, 6, 2, 2, 16)
        with pytest.raises(ValueError, match="cos and sin"):
            ops.rope_qkv(q, q, q, None, None, None, cos, sin, 6, 2, 2, 16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):     # long enough: the next check
        ops.rope(q, q, table, table, 6, 2, 2, 16)


def test_pointers_off_their_types_are_refused():
    """Each array moved off its element's boundary in turn, which a kernel would fault on."""
    lib = N.lib()
    rows = [FAKE, 0, 2, 3, 300, 100, 100]

    def each(name, args, places):
        for i, by in places:
            moved = list(args)
            moved[i] = FAKE + by
            assert getattr(lib, name)(*moved) == N.LEMA_ERR_MISALIGNED, (name, i)

    lp = rows + [FAKE, -100, 1.0, FAKE, None, None]
    each("lema_token_logprobs", lp, [(0, 1), (7, 4), (10, 2)])
    each("lema_token_logprobs", [FAKE, 1] + lp[2:], [(0, 2)])       # fp32 logits
    bwd = rows + [FAKE, -100, 1.0, FAKE, FAKE, FAKE, FAKE, 300, 100, None]
    each("lema_token_logprobs_bwd", bwd, [(0, 1), (7, 4), (11, 2), (12, 1), (13, 1)])
    each("lema_token_logprobs_bwd", [FAKE, 1] + bwd[2:], [(13, 2)])
    pref = rows + [FAKE, -100, FAKE, 0.1, 0.0, 1.0, FAKE, 1 << 20, FAKE, FAKE, FAKE, FAKE, FAKE,
                   FAKE, 300, 100, None]
    each("lema_preference_loss", pref, [(0, 1), (7, 4), (9, 2), (15, 1), (17, 3), (18, 2), (19, 1),
                                        (20, 1)])
    pol = rows + [FAKE, -100, 1.0, FAKE, FAKE, 3, 1, FAKE, 0.2, 0.2, 0.0, 0, 1.0, FAKE, 1 << 20,
                  FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 300, 100, None]
    each("lema_policy_loss", pol, [(0, 1), (7, 4), (10, 2), (11, 1), (14, 2), (22, 3), (24, 1),
                                   (25, 2), (26, 1), (27, 1)])
    dist = rows + [FAKE, 0, FAKE, 1, 3, None, 1.0, 1.0, FAKE, FAKE, 1 << 20, FAKE, FAKE, 300, 100,
                   None]
    each("lema_distill_loss", dist, [(0, 1), (7, 4), (9, 2), (15, 1), (18, 2), (19, 1)])
    ids32, tl16 = list(dist), list(dist)
    ids32[8], tl16[10] = 1, 0
    each("lema_distill_loss", ids32, [(7, 2)])
    each("lema_distill_loss", tl16, [(9, 1)])


def test_scores_refuse_a_reference_that_has_been_trained():
    from types import SimpleNamespace
    from lema_b200.trainer import StreamedLoraTrainer

    class Reached(Exception):
        pass

    def check():
        raise Reached
    ids = torch.zeros(2, 8, dtype=torch.int64)
    errors = SimpleNamespace(check=check)            # what comes next
    stepped = SimpleNamespace(layer_steps={1: 1})
    with pytest.raises(RuntimeError, match="full fine-tuning"):
        StreamedLoraTrainer.token_logprobs(
            SimpleNamespace(seq=8, full_ft=stepped, errors=errors), ids, adapters=False)
    for ft, adapters in ((stepped, True), (SimpleNamespace(layer_steps={}), False), (None, False)):
        with pytest.raises(Reached):
            StreamedLoraTrainer.token_logprobs(
                SimpleNamespace(seq=8, full_ft=ft, errors=errors), ids, adapters=adapters)


def test_kernels_that_overlap_the_one_before_wait_before_they_end():
    """A kernel that may begin while its predecessor runs must not end before that does, or
    what comes next on the stream follows this one alone: each such kernel waits, at least in
    one CTA, before any of its threads may return. Read from the sources, since the order is
    otherwise a matter of chance."""
    import re
    from lema_b200 import build
    seen = 0
    for path in build.sources():
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for body in text.split("__global__")[1:]:
            wait = body.find("griddep_wait()")
            if wait < 0:
                continue
            seen += 1
            # threads behind the last piece of work are never all of a CTA that waits
            body = re.sub(r"if \(unit >= [^;]*\) return;", "", body)
            wait = body.find("griddep_wait()")
            first = re.search(r"\breturn\b", body)
            assert first is None or wait < first.start(), (path.name, body[:120])
    assert seen >= 10
