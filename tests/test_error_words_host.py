"""What the host tells of the two error words on the device, and what goes back to zero with it."""
from conftest import compile_and_run

CHECK = r"""
#include "error_words.h"
#include <cstdio>
#include <cstring>
#include <string>
using namespace tb;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main() {
    CHECK(error_report({0, 0}, true).code == 0);
    // a failed wait is told first, whatever came behind it, and keeps the argument's code for the next time
    for (bool arguments : {false, true}) {
        const ErrorReport r = error_report({74, 75}, arguments);
        CHECK(r.code == 74 && r.wait && r.tickets && r.word == 0);
    }
    // an argument's code is told by who tells of arguments, and clears nothing but itself
    CHECK(error_report({0, 75}, false).code == 0);
    const ErrorReport r = error_report({0, 75}, true);
    CHECK(r.code == 75 && !r.wait && !r.tickets && r.word == 4);
    // the words lie in front of the tickets
    CHECK(sizeof(ErrorWords) <= kErrorTickets && kErrorTickets < kErrorBytes);
    for (int code : {71, 72, 75, 76, 81}) CHECK(std::strlen(argument_error(code)) > 20);
    CHECK(std::string(argument_error(71)) != argument_error(72) && std::string(argument_error(75)) != argument_error(71));
    puts("ok");
    return 0;
}
"""


def test_a_failed_wait_is_told_first_and_an_argument_clears_nothing_else(tmp_path):
    assert compile_and_run(tmp_path, CHECK).strip() == "ok"
