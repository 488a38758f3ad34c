"""The tags a grammar takes from a context's tables against what the line ingest keeps of them, as the oracle says it: host code, no GPU."""
import json
import random

import pytest

from helpers import Config, Oracle, shipped_config
from reply_plain import PlainGrammar
from test_replies_cpu import check_against_plain, compiled, sim  # noqa: F401

BYTES = [bytes([b]) for b in range(256)] + [b""]


def grammar_tags(g):
    """The compiled grammar's tags as they are written: over a list of the single bytes every entry of a place is one byte on, so the texts
    of the places are walked from the empty one."""
    text, todo, tags = {0: b""}, [0], set()
    end, after = g["info"].n_prefixes + 1, g["info"].n_prefixes
    while todo:
        at = todo.pop()
        for e in range(int(g["begin"][at]), int(g["begin"][at + 1])):
            to, token = int(g["move"][e]) & 0x3FFFFFFF, int(g["token"][e])
            if to == end:
                tags.add(text[at].decode())
            elif to != after and to not in text:
                text[to] = text[at] + bytes([token])
                todo.append(to)
    return tags


def kept_by_the_ingest(oracle, tag):
    """Whether a line of this tag is taken, the tag in whatever form it has by then is selected, and that form is in the vocabulary."""
    line = ", ".join([tag] * 3)                                # two commas: without them a line of one long tag looks bad
    if not oracle.normalize_raw_tag_line(line):
        return False
    selected = tag
    for _ in range(3):                                          # the line's parts, the candidates, the selected tags (Program.cs:599, 629, 694)
        selected = oracle.normalize_tag(selected)
    return selected in oracle.select_tags_from_line(line) and not (oracle.info.known_found and oracle.run_texts([line], detail=True).details[0]["unknown"].count(selected))


def written(tag, spaces):
    return tag.replace("_", " ") if spaces else tag


def check_tags(sim, vocabulary, spaces=0, **kw):  # noqa: F811
    """The grammar's tags are those of the vocabulary that ShouldDropTag lets pass as they stand there, and that the ingest keeps; returns them and the rest."""
    kw["vocabulary"] = "\n".join(vocabulary).encode()
    g, oracle = compiled(sim, BYTES, 256, tables=Config(**kw), spaces=spaces), Oracle(Config(**kw))
    assert not isinstance(g, str), g
    got = grammar_tags(g)
    kept = {t for t in vocabulary if not oracle.should_drop_tag(t) and kept_by_the_ingest(oracle, written(t, spaces))}
    assert got == {written(t, spaces) for t in kept}
    check_against_plain(g, PlainGrammar(sorted(kept), BYTES, 256, spaces=bool(spaces)))
    return kept, set(vocabulary) - kept


def lexicon(aliases):
    return json.dumps({"aliases": aliases}).encode()


@pytest.mark.parametrize("spaces", [0, 1])
def test_aliases_lead_to_kept_tags(sim, spaces):  # noqa: F811
    words = ["blond_hair", "solo", "smile", "hat"]
    alias = dict(lexicon=lexicon({"blond_hair": "blonde_hair"}))
    assert check_tags(sim, words, spaces, **alias)[1] == {"blond_hair"}                                       # an alias of a tag that is not in the vocabulary
    assert check_tags(sim, words + ["blonde_hair"], spaces, **alias)[1] == set()                              # of one that is
    assert check_tags(sim, words + ["blonde_hair"], spaces, denylist=b"blonde_hair", **alias)[1] == {"blond_hair", "blonde_hair"}   # of a denied one
    assert check_tags(sim, words + ["watermark"], spaces, lexicon=lexicon({"hat": "watermark"}))[1] == {"hat", "watermark"}         # of one that the pipeline drops
    assert check_tags(sim, words + ["x"], spaces, lexicon=lexicon({"hat": "x"}))[1] == {"hat", "x"}           # of one letter
    assert check_tags(sim, words + ["hat,smile"], spaces, lexicon=lexicon({"hat": "hat,smile"}))[1] == {"hat", "hat,smile"}   # of what is no tag


def test_every_hop_counts(sim):  # noqa: F811
    words = ["a1", "b1", "c1", "d1", "solo", "smile"]
    chain = dict(lexicon=lexicon({"a1": "b1", "b1": "c1", "c1": "d1"}))
    assert check_tags(sim, words, **chain)[1] == set()
    assert check_tags(sim, words, denylist=b"d1", **chain)[1] == {"a1", "b1", "c1", "d1"}       # the third hop is the selected tag's
    assert check_tags(sim, words, denylist=b"b1", **chain)[1] == {"a1", "b1"}
    assert check_tags(sim, ["a1", "b1", "c1", "solo"], **chain)[1] == {"a1", "b1", "c1"}        # they end in a tag that is not in the vocabulary
    circle = dict(lexicon=lexicon({"a1": "b1", "b1": "a1"}))
    assert check_tags(sim, words, **circle)[1] == set()
    assert check_tags(sim, words, denylist=b"b1", **circle)[1] == {"a1", "b1"}
    assert check_tags(sim, ["a1", "solo"], **circle)[1] == {"a1"}


def test_tables_without_a_vocabulary(sim):  # noqa: F811
    """Every tag of the built-in tables is kept, alias keys among them; of a lexicon's an alias of a denied one is not."""
    kw = dict(lexicon=lexicon({"hat": "bad_hat", "cap": "hood"}), denylist=b"bad_hat")
    tags, oracle = grammar_tags(compiled(sim, BYTES, 256, tables=Config(**kw))), Oracle(Config(**kw))
    assert "soles" in tags and {"cap", "hood"} <= tags and not {"hat", "bad_hat"} & tags
    for t in tags:
        assert kept_by_the_ingest(oracle, t), t


def test_shipped_tables(sim):  # noqa: F811
    tags, oracle = grammar_tags(compiled(sim, BYTES, 256, tables=shipped_config())), Oracle(shipped_config())
    assert len(tags) > 5000
    for t in sorted(tags)[::7]:
        assert kept_by_the_ingest(oracle, t), t


PHRASES = ["unable_to_stand", "has_an_airplane", "i_cannot", "hawaii_can't_swim", "cannot_provide_hat", "i'm_not_able", "i_won't"]


@pytest.mark.parametrize("spaces", [0, 1])
def test_no_phrase_behind_underscores(sim, spaces):  # noqa: F811
    """Most phrases of a refusal hold blanks: a tag that spells one with them has the whole line refused."""
    words = ["solo", "smile", "long_hair", "sorry_face", "unable"]
    assert check_tags(sim, words + PHRASES, spaces)[1] == {"sorry_face"} | (set(PHRASES) if spaces else set())
    oracle = Oracle(Config(vocabulary="\n".join(words + PHRASES).encode()))
    for t in PHRASES:
        assert bool(oracle.normalize_raw_tag_line(", ".join([written(t, spaces), "solo", "smile"]))) == (not spaces), t


def test_a_tag_that_cannot_be_written_with_spaces(sim):  # noqa: F811
    """A blank at a tag's end is trimmed off: the context's tags that end in one are left out, a caller's are refused by name."""
    words = ["solo_", "solo", "smile", "hat_(a)_", "hat_(a)"]
    assert check_tags(sim, words, 0)[1] == set()
    g = compiled(sim, BYTES, 256, tables=Config(vocabulary="\n".join(words).encode()), spaces=1)
    assert not isinstance(g, str) and grammar_tags(g) == {"solo", "smile", "hat (a)"}
    refusal = compiled(sim, BYTES, 256, tags=words, spaces=1)
    assert "ends with a space" in refusal and '"hat (a) "' in refusal or '"solo "' in refusal, refusal
    assert '"so,lo"' in compiled(sim, BYTES, 256, tags=["so,lo"])


ALIASES = {"soles": "foot_sole", "blond_hair": "blonde_hair", "hood": "watermark", "cap": "hats"}
WORDS = ["1girl", "solo", "soles", "foot_sole", "blond_hair", "blonde_hair", "blue_eyes", "hood", "cap", "hats", "unable_to_stand", "long_hair", "smile", "a_", "school_uniform", "blue_sky"]


@pytest.mark.parametrize("spaces", [0, 1])
def test_finished_lines_are_taken(sim, spaces):  # noqa: F811
    """Lines of at least three of the grammar's tags, repeats among them: none is refused, and every different tag is selected and known."""
    cfg = Config(vocabulary="\n".join(WORDS).encode(), lexicon=lexicon(ALIASES), trigger="solo")
    oracle, rng = Oracle(cfg), random.Random(11)
    tags = sorted(grammar_tags(compiled(sim, BYTES, 256, tables=cfg, spaces=spaces)))
    assert set(WORDS) - {t.replace(" ", "_") for t in tags} == {"hood", "soles"} | ({"unable_to_stand", "a_"} if spaces else set())   # the vocabulary has read "soles" as "foot_sole"
    lines = [[rng.choice(tags) for _ in range(rng.randint(3, 12))] for _ in range(300)]
    got = oracle.run_texts([", ".join(line) for line in lines], detail=True)
    assert got.counters["line_rejected"] == 0 and not got.verdicts["n_dropped"].any()
    for line, v, d in zip(lines, got.verdicts, got.details):
        kept = {oracle.normalize_tag(t) for t in line}
        selected = oracle.select_tags_from_line(", ".join(line))
        assert v["n_candidates"] == len(kept) and set(selected) == kept | {"1girl", "solo"} and len(selected) == v["n_selected"]
        assert not kept & set(d["unknown"])
        assert bool(v["flags"] & 0x08) == (len(selected) < 3)                    # the fallback


def test_what_a_finished_line_may_still_be(sim):  # noqa: F811
    """What the header does not promise: repeats count as written tags, two tags of more than 40 characters are refused, and a caption ends at 42 tags."""
    words = ["1girl", "sgrui", "blue_eyes", "a" * 25, "b" * 25] + ["w%d" % k for k in range(60)]
    oracle = Oracle(Config(vocabulary="\n".join(words).encode()))
    assert oracle.select_tags_from_line("blue_eyes, blue_eyes, blue_eyes") == ["sgrui", "1girl", "blue_eyes"]
    assert oracle.run_texts(["1girl, sgrui, 1girl", "%s, %s" % (words[3], words[4]), "%s, 1girl" % words[3], "%s, %s, 1girl" % (words[3], words[4])]).verdicts["flags"].tolist() == [0x09, 0x19, 0x01, 0x01]
    long = oracle.select_tags_from_line(", ".join(words[5:47]))
    assert len(long) == 42 and long[:2] == ["sgrui", "1girl"] and len(set(long) & set(words[5:47])) == 40
