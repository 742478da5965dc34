"""Generation with drafted tokens against generation without: the same tokens, in fewer passes where the guesses are right."""
import random
import subprocess
import sys

import pytest
import torch

import plain_gpt2
from helpers import PAGE_SIZE, ROOT, make_model, oracle_store, random_ids
from test_generate_gpu import follow

pytestmark = pytest.mark.gpu
STORE = {"float32": torch.float32, "bfloat16": torch.bfloat16}


@pytest.fixture(scope="module", params=[("A", "float32"), ("B", "float32"), ("C", "float32"), ("A", "bfloat16"), ("C", "bfloat16")],
                ids=lambda p: f"{p[0]}-{p[1]}")
def setup(request, tmp_path_factory):
    which, dtype = request.param
    d = str(tmp_path_factory.mktemp(f"draft_{which}_{dtype}"))
    make_model(d, which, seed=31, dtype=STORE[dtype])
    cfg, w = plain_gpt2.read_model(d)
    return dict(which=which, dtype=dtype, dir=d, cfg=cfg, w=w, page=PAGE_SIZE[which])


def make(setup, **kw):
    import mini_llm_b200 as m
    args = dict(dtype=setup["dtype"], page_size=setup["page"], max_tokens=4096, max_num_seqs=4, max_num_batched_tokens=64, prefill_chunk=24)
    args.update(kw)
    return m.LLM(setup["dir"], **args)


class Knowing:
    """Drafts the tokens that are known to follow (``answers``: prompt -> tokens), after wrong guesses that stand before them."""

    def __init__(self, answers, vocab, right=True):
        self.answers, self.vocab, self.right, self.rng = answers, vocab, right, random.Random(5)

    def draft(self, tokens, rows, depth):
        whole = next(a for p, a in self.answers.items() if tuple(tokens[:len(p)]) == p)
        coming = whole[len(tokens):]
        out, parents = [tokens[-1]], [-1]
        at = 0
        for k in range(min(depth - 1, len(coming))):
            for _ in range(self.rng.randrange(2)):
                if len(out) < rows - 1:
                    out.append(self.rng.randrange(self.vocab))
                    parents.append(at)
            if len(out) >= rows:
                break
            out.append(coming[k] if self.right else (coming[k] + 1) % self.vocab)
            parents.append(at)
            at = len(out) - 1
        return out, parents


def check(setup, prompts, got, limit, what):
    for p, o in zip(prompts, got):
        follow(setup["cfg"], setup["w"], p, o, oracle_store(setup["dtype"]), limit, what, setup["dtype"])


@pytest.mark.parametrize("rows,depth", [(1, 1), (8, 4), (16, 8), (33, 12)])
def test_the_same_tokens_as_without_drafts(setup, rows, depth):
    import mini_llm_b200 as m
    prompts = [random_ids(n, setup["cfg"]["vocab_size"], 7 + n) for n in (5, 17, 32, 1, 40)]
    sp = m.SamplingParams(max_new_tokens=20, ignore_eos=True)
    want = make(setup).generate(prompts, sp)
    answers = {tuple(p): list(p) + w for p, w in zip(prompts, want)}
    llm = make(setup)
    for drafter in (None, Knowing(answers, setup["cfg"]["vocab_size"]), Knowing(answers, setup["cfg"]["vocab_size"], right=False)):
        got = llm.generate_drafted(prompts, sp, drafter=drafter, rows=rows, depth=depth)
        assert all(len(o) == 20 for o in got)
        if setup["dtype"] == "float32":
            assert got == want
        else:
            check(setup, prompts, got, 0.15, f"drafts of {rows} rows")
        assert llm.runner.cache.num_live == 0
        llm.runner.cache.check()
        if isinstance(drafter, Knowing) and drafter.right and depth >= 4 and setup["dtype"] == "float32":
            assert llm.draft_stats.tokens >= 2 * llm.draft_stats.requests        # the right guesses were kept


def test_temperature_draws_the_same_tokens(setup):
    import mini_llm_b200 as m
    prompts = [random_ids(n, setup["cfg"]["vocab_size"], 70 + n) for n in (1, 9, 40)]
    params = [m.SamplingParams(temperature=t, seed=1234, max_new_tokens=14, ignore_eos=True) for t in (0.8, 0.0, 1.3)]
    llm = make(setup)
    want = llm.generate(prompts, params)
    answers = {tuple(p): list(p) + w for p, w in zip(prompts, want)}
    other = make(setup)                                   # request numbers from 0 again: the same draws
    got = other.generate_drafted(prompts, params, drafter=Knowing(answers, setup["cfg"]["vocab_size"]), rows=12, depth=6)
    if setup["dtype"] == "float32":
        assert got == want
    else:
        assert [len(o) for o in got] == [14] * 3


def test_to_the_end_of_the_context(setup):
    """Every position is fed once, and one token more comes out, whatever the drafts' depth."""
    import mini_llm_b200 as m
    P = setup["cfg"]["n_positions"]
    prompt = random_ids(P - 45, setup["cfg"]["vocab_size"], 5)
    sp = m.SamplingParams(max_new_tokens=10 * P, ignore_eos=True)
    want = make(setup).generate([prompt], sp)[0]
    got = make(setup).generate_drafted([prompt], sp, drafter=Knowing({tuple(prompt): prompt + want}, setup["cfg"]["vocab_size"]))[0]
    assert len(got) == 46
    if setup["dtype"] == "float32":
        assert got == want


def test_the_end_of_sequence_token_ends_a_request_within_a_path(setup):
    import mini_llm_b200 as m
    prompts = [random_ids(n, setup["cfg"]["vocab_size"], 40 + n) for n in (6, 11)]
    free = make(setup).generate(prompts, m.SamplingParams(max_new_tokens=16, ignore_eos=True))
    llm = make(setup)
    llm.runner.spec.eos_token_id = free[0][9]
    answers = {tuple(p): list(p) + w for p, w in zip(prompts, free)}
    got = llm.generate_drafted(prompts, m.SamplingParams(max_new_tokens=16), drafter=Knowing(answers, setup["cfg"]["vocab_size"]), rows=12)
    if setup["dtype"] == "float32":
        for o, f in zip(got, free):
            cut = f.index(free[0][9]) + 1 if free[0][9] in f else 16
            assert o == f[:cut]


def test_a_pool_for_one_request_at_a_time(setup):
    """Requests wait for pages; one that can never fit is refused and leaves nothing behind."""
    import mini_llm_b200 as m
    page = setup["page"]
    prompts = [random_ids(n, setup["cfg"]["vocab_size"], 300 + n) for n in (20, 33, 12)]
    sp = m.SamplingParams(max_new_tokens=12, ignore_eos=True)
    llm = make(setup, max_tokens=None, num_pages=-(-(33 + 12 + 8) // page) + 1)
    got = llm.generate_drafted(prompts, sp, rows=8, depth=4)
    if setup["dtype"] == "float32":
        assert got == make(setup).generate(prompts, sp)
    from mini_llm_b200.engine.runner import OutOfPages
    with pytest.raises(OutOfPages, match="no pages"):
        llm.generate_drafted([random_ids(100, setup["cfg"]["vocab_size"], 1)], sp, rows=8, depth=4)
    assert llm.runner.cache.num_live == 0
    llm.runner.cache.check()


def test_steps_of_one_shape_are_replayed_as_graphs(setup):
    import mini_llm_b200 as m
    prompts = [random_ids(9, setup["cfg"]["vocab_size"], s) for s in (1, 2)]
    llm = make(setup)
    llm.generate_drafted(prompts, m.SamplingParams(max_new_tokens=24, ignore_eos=True), rows=8, depth=4)
    # the first step with two requests and the first with one run as they come, and once more each where that brought a new buffer
    # (which drops the graphs); every other step is a graph
    assert llm.draft_stats.steps > 5 and llm.runner.graph_replays >= llm.draft_stats.steps - 4


def test_steps_stay_graphs_from_call_to_call(setup):
    """A second call replays what the first one captured; one with other rows or depths, or steps of plain decoding in between, changes
    neither call's tokens."""
    import mini_llm_b200 as m
    prompts = [random_ids(9, setup["cfg"]["vocab_size"], s) for s in (3, 4)]
    sp = m.SamplingParams(max_new_tokens=20, ignore_eos=True)
    llm = make(setup)
    want = [llm.generate_drafted(prompts, sp, rows=8, depth=d) for d in (4, 8)]
    for _ in range(3):
        llm.generate(prompts, sp)
    for d, w in ((8, want[1]), (8, want[1]), (4, want[0]), (4, want[0]), (8, want[1])):
        assert llm.generate_drafted(prompts, sp, rows=8, depth=d) == w
    before = llm.runner.graph_replays
    assert llm.generate_drafted(prompts, sp, rows=8, depth=8) == want[1]
    assert llm.runner.graph_replays - before >= llm.draft_stats.steps


def test_two_runners_of_trees_on_one_model(setup):
    """Each has buffers of its own: the one's captured steps are not the other's, whatever they have in common."""
    from mini_llm_b200.engine.drafting import DraftEntry, DraftRunner
    from mini_llm_b200.engine.runner import StepEntry
    got = {}
    for order in ("one", "both"):
        llm = make(setup)
        r = llm.runner
        runners = [DraftRunner(r, 4, 4) for _ in range(2)]
        r.add_request("q")
        r.step([StepEntry("q", random_ids(7, setup["cfg"]["vocab_size"], 5), ())])
        out, last = [], 1
        for i in range(12):
            res = runners[i % 2 if order == "both" else 0].step([DraftEntry("q", [last, last, 2, 3], [-1, 0, 1, 2])])[0]
            out += res.tokens
            last = res.tokens[-1]
        got[order] = out
    assert got["one"] == got["both"]


def test_refusals(setup, tmp_path):
    import mini_llm_b200 as m
    from mini_llm_b200.engine.drafting import DraftEntry, DraftRunner
    from mini_llm_b200.engine.runner import StepError
    llm = make(setup)
    rid = llm.add_request([1, 2, 3])
    with pytest.raises(RuntimeError, match="unfinished"):
        llm.generate_drafted([[1, 2]])
    llm.abort(rid)
    for prompt in ([], [setup["cfg"]["vocab_size"]], [0] * (setup["cfg"]["n_positions"] + 1)):
        with pytest.raises(ValueError):
            llm.generate_drafted([prompt])
    llm.runner.add_request("r")
    trees = DraftRunner(llm.runner, 4, 4)
    for e, words in ((DraftEntry("r", [1] * 5, [-1] * 5), "rows are taken"), (DraftEntry("r", [1, 2], [-1]), "parents"),
                     (DraftEntry("r", [1, 2], [-1, 1]), "come before"), (DraftEntry("r", [1, -4], [-1, 0]), "vocabulary"),
                     (DraftEntry("q", [1], [-1]), "not live"), (DraftEntry("r", [1, 2], [-1, 0], 0.5, [0.1]), "uniform")):
        with pytest.raises(StepError, match=words):
            trees.step([e])
    with pytest.raises(StepError, match="twice"):
        trees.step([DraftEntry("r", [1], [-1])] * 2)
    llm.runner.finish_request("r")


def test_a_model_whose_layers_carry_a_state_is_refused(tmp_path):
    import mini_llm_b200 as m
    from mini_llm_b200.engine.runner import StepError
    from helpers import write_model
    from test_zanelorn_gpu import CONFIGS as STATES, make_tensors
    which = next(iter(STATES))
    d = write_model(str(tmp_path), STATES[which], make_tensors(STATES[which], seed=3), torch.float32)
    llm = m.LLM(d, dtype="float32", max_tokens=512, max_num_seqs=2)
    with pytest.raises(StepError, match="drafts need"):
        llm.generate_drafted([[1, 2, 3]])


def test_the_command_line(setup):
    cmd = [sys.executable, "-m", "mini_llm_b200", "--model", setup["dir"], "--dtype", setup["dtype"], "--page-size", str(setup["page"]),
           "--num-pages", "64", "--max-new-tokens", "9", "--ignore-eos", "--prompt-ids", "5 6 7 5 6", "--prompt-ids", "11"]
    plain = subprocess.run(cmd, cwd=ROOT, capture_output=True, text=True, timeout=300)
    drafted = subprocess.run(cmd + ["--draft-rows", "8", "--stats"], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert plain.returncode == 0 and drafted.returncode == 0, drafted.stderr
    assert '"steps"' in drafted.stderr
    if setup["dtype"] == "float32":
        assert drafted.stdout == plain.stdout
    assert subprocess.run(cmd + ["--draft-rows", "8", "--stream"], cwd=ROOT, capture_output=True, timeout=300).returncode == 1
