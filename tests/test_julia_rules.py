"""CPU: the ChainRules rules of the vocabulary operators, read as text (the Julia sources cannot be executed here)."""
import re
from pathlib import Path

TYLO = Path(__file__).resolve().parent.parent / "tylo.jl_b200" / "julia" / "Tylo"
RULES = (TYLO / "ext" / "ChainRulesCoreExt.jl").read_text()


def body(text, opening):
    """A top-level function, from `opening` to the `end` in the first column."""
    at = text.index(opening)
    return text[at:text.index("\nend", at)]


def rule(name):
    return re.sub(r"#.*", "", body(RULES, f"function rrule(::typeof({name})"))


def test_every_result_of_the_scores_has_its_cotangent_looked_at():
    """A field of the result whose cotangent the pullback never reads would drop a gradient without a word."""
    primal = body((TYLO / "src" / "vocab" / "logprobs.jl").read_text(), "function token_logprobs(")
    fields = [f.split("=")[0].strip() for f in re.search(r"return \(;\s*(.*)\)", primal).group(1).split(",")]
    assert fields == ["logp", "entropy", "top"]
    for f in fields:
        assert f"Ȳ.{f}" in rule("token_logprobs"), f
    assert "throw(ArgumentError(" in rule("token_logprobs")        # the alternatives' cotangent, which has no kernel


def keywords(signature):
    """Names of the keyword arguments of a one-line function signature; splats keep their dots."""
    inside = signature[signature.index(";") + 1:signature.rindex(")")]
    return {k.split("=")[0].strip() for k in inside.split(",")}


def test_the_rule_takes_the_keywords_of_the_operator():
    source = (TYLO / "src" / "vocab" / "logprobs.jl").read_text()
    assert keywords(rule("token_logprobs").split("\n")[0]) == keywords(body(source, "function token_logprobs(").split("\n")[0])


def test_checkpoints_given_by_the_caller_reach_forward_and_backward():
    for name in ("token_logprobs", "distill"):
        text = rule(name)
        assert "checkpoints = nothing" in text.split("\n")[0], name
        assert "cp = checkpoints === nothing ?" in text, name
        assert text.count("checkpoints = cp") == 2, name


def test_a_loss_that_is_not_used_has_a_zero_gradient():
    """The pullback may be handed a zero tangent, which has no memory to give to a kernel."""
    for name in ("token_logprobs", "distill"):
        pullback = rule(name)[rule(name).index("pullback("):]
        assert "isa AbstractZero" in pullback[:pullback.index("∇" + name)], name
