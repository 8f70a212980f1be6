"""Every assembly statement of the kernels says which fixed registers it writes: the compiler may keep a value of its
own in a register that a statement does not name."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STATEMENT = re.compile(r"\basm\s+volatile\s*\((.*?)\);", re.S)
STRING = r'"(?:[^"\\]|\\.)*"'


def statements():
    for path in sorted(glob.glob(os.path.join(ROOT, "anni_amd", "csrc", "*.h*"))):
        text = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
        for body in STATEMENT.findall(text):
            template = re.match(r"\s*((?:%s\s*)+)" % STRING, body).group(1)
            # template : outputs : inputs : clobbers
            depth, lists, last = 0, [], 0
            rest = body[len(template):]
            quoted = [m.span() for m in re.finditer(STRING, rest)]
            for k, ch in enumerate(rest):
                if any(a <= k < b for a, b in quoted):
                    continue
                depth += (ch == "(") - (ch == ")")
                if ch == ":" and depth == 0:
                    lists.append(rest[last:k])
                    last = k + 1
            lists.append(rest[last:])
            clobbers = re.findall(r'"(\w+)"', lists[3]) if len(lists) > 3 else []
            yield os.path.basename(path), "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', template)), clobbers


def test_written_registers_are_named():
    seen = 0
    for name, code, clobbers in statements():
        for line in re.split(r"\\n\\t|\\n|;", code):
            words = re.split(r"[\s,]+", line.strip())
            dst = words[1] if len(words) > 1 else ""
            if re.match(r"(m0|vcc\w*|exec\w*|s\d+|s\[\d|v\d+|v\[\d)", dst) and not words[0].startswith(("s_cmp", "global_store")):
                seen += 1
                assert dst in clobbers, (name, line, clobbers)
    assert seen >= 1            # the load into LDS, which takes its place from m0
