"""A type or function of external linkage has one definition: no two of the library's sources define one of the same qualified name (the linker would keep either of
two inline ones, and an instance of a template on two types of one name would be one of two)."""
import os
import re

from anode_b200 import build

TEXT = re.compile(r'//[^\n]*|/\*.*?\*/|"(?:\\.|[^"\\\n])*"|\'(?:\\.|[^\'\\\n])+\'', re.S)
DIRECTIVE = re.compile(r"^[ \t]*#(?:[^\n]*\\\n)*[^\n]*$", re.M)


def definitions(source):
    """Qualified names of the types and functions with a body that a source defines at namespace scope, but for static ones, those in unnamed namespaces and those of C."""
    source = DIRECTIVE.sub("", TEXT.sub(lambda m: '"C"' if m.group() == '"C"' else " ", source))
    names, spaces, depth, start = set(), [], 0, 0          # depth: braces that are no namespaces
    for at in re.finditer(r"[{};]", source):
        c, head = at.group(), source[start:at.start()].strip()
        if depth == 0 or c != ";":
            start = at.end()
        if c == "{" and depth == 0:
            if re.fullmatch(r"(inline )?namespace(\s+[\w:]+)?", head):
                spaces.append(head.split()[-1] if head != "namespace" else None)
                continue
            if head == 'extern "C"':
                spaces.append(None)
                continue
            head = re.sub(r"^(template\s*<[^{}]*?>\s*(?=\b(?:struct|class|__global__|__device__|__host__|inline|static|constexpr|void|int|bool|auto|typename|const|uint|float)))+", "", head)
            type_ = re.match(r"(?:struct|class|union|enum(?:\s+class)?)\s+(?:__align__\(\d+\)\s+|alignas\(\d+\)\s+)?(\w+)\s*(?:final\s*)?(?::[^:].*)?$", head, re.S)
            function = None if type_ or "=" in head.split("(")[0] else re.search(r"(\w+)\s*\(", re.sub(r"__launch_bounds__\s*\((?:[^()]|\([^()]*\))*\)|alignas\(\w+\)", "", head))
            found = type_ or function
            if found and None not in spaces and not re.search(r'\bstatic\b|extern "C"', head):
                names.add("::".join(spaces + [found.group(1)]))
            depth = 1
        elif c == "{":
            depth += 1
        elif c == "}":
            if depth:
                depth -= 1
            else:
                spaces.pop()
    assert not spaces and depth == 0
    return names


def test_the_reader_of_sources():
    text = """
    #define X {
    namespace a { struct S { int f() { return 1; } }; /* struct No {}; */ template <typename T> struct V { T v; };
    template <typename T, int N> __global__ void __launch_bounds__(most(N), 2) k(const S s) { if (s.x) { y(); } } inline bool g(int a) { return "{"; }
    static int h() { return 0; } namespace { int i() { return 0; } struct H {}; } constexpr int n = 3; int declared(int); struct Declared; namespace b { struct S : V<int> {}; } }
    extern "C" int c(int a) { return a; }
    extern "C" { int d() { return 1; } }
    """
    assert definitions(text) == {"a::S", "a::V", "a::k", "a::g", "a::b::S"}


def test_no_two_sources_define_one_name():
    where = {}
    for name in build.SOURCES:
        with open(os.path.join(build.CSRC, name)) as f:
            for d in definitions(f.read()):
                where.setdefault(d, []).append(name)
    assert len(where) > 100
    assert not {d: files for d, files in where.items() if len(files) > 1}
