"""One name, one type: no two translation units of the library define a struct, class or
enumeration of the same qualified name (they are linked together)."""
import collections
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-darwinml_amd", "csrc")

TYPE = re.compile(r"\b(?:struct|class|union|enum(?:\s+class)?)\s+(\w+)\s*(<[^;{}]*>)?\s*(?:final)?\s*(?::[^:].*)?$", re.S)


def types(text, unit):
    """The qualified names of the types that `text` defines at namespace scope."""
    text = re.sub(r'R"(\w*)\(.*?\)\1"', '""', text, flags=re.S)
    text = re.sub(r'//[^\n]*|/\*.*?\*/|"(?:\\.|[^"\\\n])*"|\'(?:\\.|[^\'\\\n])\'', " ", text, flags=re.S)
    names, scopes, last = [], [], 0
    for m in re.finditer(r"[{};]", text):
        head, last = text[last:m.start()].strip(), m.end()
        if m.group() == "}" and scopes:
            scopes.pop()
        if m.group() != "{":
            continue
        space, kind = re.search(r"\bnamespace\s*([\w:]*)$", head), TYPE.search(head)
        if space:
            scopes.append(space.group(1) or f"(unnamed in {unit})")
        elif re.search(r"\bextern\s*$", head):  # extern "C", its string gone
            scopes.append("")
        else:
            if kind and None not in scopes:
                names.append("::".join([s for s in scopes if s] + [kind.group(1) + re.sub(r"\s", "", kind.group(2) or "")]))
            scopes.append(None)
    return names


def test_types():
    """What types() reads."""
    text = """namespace a { struct S { struct In {}; }; template <int N> struct T {}; template <> struct T<2> : S {};
    namespace { class C { void f() { struct L {}; } }; } struct Fwd; extern "C" { enum E { x }; } }  // struct Not {
    struct S { int a; };"""
    assert types(text, "f") == ["a::S", "a::T", "a::T<2>", "a::(unnamed in f)::C", "a::E", "S"]


def test_no_name_is_defined_twice():
    where = collections.defaultdict(set)
    for path in sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.cpp"))):
        with open(path) as f:
            for name in types(f.read(), os.path.basename(path)):
                where[name].add(os.path.basename(path))
    assert len(where) > 20
    assert not {n: sorted(w) for n, w in where.items() if len(w) > 1}
