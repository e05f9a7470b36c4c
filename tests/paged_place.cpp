// Answers the arithmetic of blok_amd/csrc/kx_paged_place.h: lines of a letter and numbers on stdin.
#include <stdio.h>
#include <string.h>
#include "kx_paged_place.h"

int main() {
  char what;
  while (scanf(" %c", &what) == 1) {
    if (what == 'r') {
      int from, to, pos, tokens, cap;
      if (scanf("%d %d %d %d %d", &from, &to, &pos, &tokens, &cap) != 5) return 1;
      const kxpage::Rows r = kxpage::rows_of(from, to, pos, tokens, cap);
      printf("%d %d %d %d %d\n", r.first, r.n, r.pos, r.fault, kxpage::units_of(r.pos, r.n));
    } else if (what == 'g') {
      int id, pages;
      if (scanf("%d %d", &id, &pages) != 2) return 1;
      printf("%d\n", kxpage::page_ok(id, pages));
    } else if (what == 'p') {
      int t;
      if (scanf("%d", &t) != 1) return 1;
      printf("%d %d\n", kxpage::place_of(t), kxpage::token_of(t));
    } else if (what == 'e') {
      float x;
      if (scanf("%a", &x) != 1) return 1;
      uint32_t u;
      memcpy(&u, &x, 4);
      const int e = kxpage::exponent_of(u);
      printf("%d %d\n", e, kxpage::scale_exponent(kxpage::scale_bits(e)));
    } else if (what == 'w') {
      int k, v;
      if (scanf("%d %d", &k, &v) != 2) return 1;
      const kxpage::Widths w = kxpage::widths_of(k, v);
      printf("%d %d\n", w.k, w.v);
    }
  }
}
